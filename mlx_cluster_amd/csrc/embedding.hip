// Embedding lookup with scaling, and its gradient by sorted nodes: the rows of
// a walk's nodes, and their way back.
//
//   lookup     y[i, :] = s * W[x_i, :]
//   gradient   G[v, :] = s * sum over i with x_i = v of g[i, :]
//
// The gradient sorts the places by node (place_sort.hip).  Walks visit hubs tens
// of thousands of times, so the sorted places are added up in tiles of 32, each
// by one group of lanes whatever runs it holds; a run that crosses tiles is put
// together from its tiles' parts, a hub's from sums of 16 tiles, of 16 of these,
// and so on.  A lane's chain of float32 additions is then 32 rows, and for a run
// that crosses tiles at most 30 parts a level and about 510 of the highest (the
// next level is built from 32 tiles on).  In lists of up to 16,384 places, which
// one launch takes, a lane adds up its share of a block's places: 8, or of hubs up to
// 1,024 (rows of more than 32 packs).  Nothing is added with atomics, and the order
// of a sum depends on the places alone.
//
// Bound by the gather of the rows and the table's stores.  2.65 M rows of 128
// bfloat16 (680 MB) into a table of 2^20 (268 MB): 318 us, of which the tiles take
// 180, the runs that cross them 36, the zeros and the sort 102.  One wavefront a
// node, place after place, took 1,530 us for the sums alone.
#include "place_sort.h"

namespace mlxc {

namespace {

// ------------------------------------------------------------- lookup

// Packs of N elements: a block takes kBlock * kAhead of them in a row, a thread
// every kBlock-th, its loads in flight together.  A pack's row is a 32-bit
// division from the block's first (a 64-bit one a pack kept the vector units busy).
//
// Bound by the rows' stream: 2.65 M rows of 128 bfloat16 (680 MB written, a table
// of 268 MB) in 183 us; 248 without kStreamed, stores past the caches.  Results
// that the caches hold for whoever reads them next are stored there, by one
// pack a thread (2,000 rows of 64: 2.8 us, 4.3 with four).
template <typename E, int N, int kAhead, bool kStreamed>
__global__ __launch_bounds__(kBlock) void embedding_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, uint32_t packs, uint32_t inverse,
    Nodes nodes, int64_t count, float scale, typename E::S* __restrict__ out, int64_t* status) {
    using S = typename E::S;
    constexpr int kChunk = kBlock * kAhead;
    const int64_t total = count * packs;
    bool bad = false;
    for (int64_t base = blockIdx.x * static_cast<int64_t>(kChunk); base < total;
         base += static_cast<int64_t>(gridDim.x) * kChunk) {
        const int64_t row0 = base / packs;  // the same in all threads
        const uint32_t rest = static_cast<uint32_t>(base - row0 * packs);
        int64_t node[kAhead];
        uint32_t d[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t e = rest + u * kBlock + threadIdx.x;
            uint32_t q = packs > 1 ? __umulhi(e, inverse) : e;
            if (q * packs > e) --q;  // the inverse is rounded up
            d[u] = (e - q * packs) * N;
            const int64_t i = row0 + q;
            node[u] = i < count ? node_at(nodes, i, bad) : -1;
        }
        Pack<S, N> x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (node[u] >= 0)
                x[u] = *reinterpret_cast<const Pack<S, N>*>(weight + node[u] * row_stride + d[u]);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t e = base + u * kBlock + threadIdx.x;
            Pack<S, N> y;
#pragma unroll
            for (int k = 0; k < N; ++k)
                y.v[k] = node[u] >= 0 ? E::store(E::load(x[u].v[k]) * scale) : S(0);
            if (e >= total) continue;
            if constexpr (kStreamed) stream_pack(out + e * N, y);
            else *reinterpret_cast<Pack<S, N>*>(out + e * N) = y;
        }
    }
    report_bad(bad, status);
}

// Rows whose packs are smaller than 16 bytes (odd sizes): a thread makes kAll =
// 16 bytes' worth of the output's elements from pieces of N, of one row and, as
// dim >= kAll, at most the next, and stores them whole.  1 M rows of 33 float32
// 99 us with a piece a thread, so 62; 2.74 M of 33 bfloat16 144 and 126.  Bound by
// the pieces' load instructions.
template <typename E, int N, bool kStreamed>
__global__ __launch_bounds__(kBlock) void embedding_odd_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, uint32_t dim, uint32_t inverse,
    Nodes nodes, int64_t count, float scale, typename E::S* __restrict__ out, int64_t* status) {
    using S = typename E::S;
    constexpr int kAll = 16 / sizeof(S);
    const int64_t total = count * dim;
    bool bad = false;
    for (int64_t base = blockIdx.x * static_cast<int64_t>(kBlock * kAll); base < total;
         base += static_cast<int64_t>(gridDim.x) * kBlock * kAll) {
        const int64_t row0 = base / dim;  // the same in all threads
        const uint32_t e = static_cast<uint32_t>(base - row0 * dim) + threadIdx.x * kAll;
        uint32_t q = __umulhi(e, inverse);
        if (q * dim > e) --q;  // the inverse is rounded up
        uint32_t d = e - q * dim;
        const int64_t i = row0 + q, at = base + threadIdx.x * kAll;
        const int64_t first = i < count ? node_at(nodes, i, bad) : -1;
        const int64_t second = i + 1 < count ? node_at(nodes, i + 1, bad) : -1;
        const S* row = weight + (first < 0 ? 0 : first) * row_stride;
        const S* next = weight + (second < 0 ? 0 : second) * row_stride;
        Pack<S, N> x[kAll / N];
        uint32_t have = 0;
#pragma unroll
        for (int k = 0; k < kAll / N; ++k) {
            const uint32_t here = d + k * N;
            const bool own = here < dim;
            // (of no node the table's first row, for a load without a branch)
            x[k] = *reinterpret_cast<const Pack<S, N>*>(own ? row + here : next + (here - dim));
            have |= static_cast<uint32_t>(own ? first >= 0 : second >= 0) << k;
        }
        Pack<S, kAll> y;
#pragma unroll
        for (int k = 0; k < kAll; ++k)
            y.v[k] = (have >> (k / N)) & 1 ? E::store(E::load(x[k / N].v[k % N]) * scale) : S(0);
        if (at + kAll <= total) {
            if constexpr (kStreamed) stream_pack(out + at, y);
            else *reinterpret_cast<Pack<S, kAll>*>(out + at) = y;
        } else {
#pragma unroll
            for (int k = 0; k < kAll; ++k)
                if (at + k < total) out[at + k] = y.v[k];
        }
    }
    report_bad(bad, status);
}

// ------------------------------------------------------------- sums

// The sorted places are added up in tiles of kSpan.  Level 1's tiles hold kFan
// of these, level l's kFan^l.
constexpr int kFan = 16;
constexpr int kMaxLevels = 6;
// A level is built where it has this many tiles: with fewer a run has few parts
// of the level below.
constexpr int64_t kLevelTiles = 32;

// The lanes that serve one row: 2^lanes_log of them, a pack of N columns each,
// from column first_column on.
struct RowShape {
    int32_t dim;
    int32_t lanes_log;
};

// acc += rows index(from) .. index(to - 1), in order; kBatch loads in flight, those
// past the end of the last row again, and added as zeros: added behind a branch,
// they are moved there by the compiler, one load after the other (a batch then
// takes 12.7 us instead of 2).
constexpr int kBatch = 8;
template <typename E, int N, typename Index>
__device__ __forceinline__ void add_rows(float (&acc)[N], const typename E::S* __restrict__ rows,
                                         int32_t dim, int32_t col, int64_t from, int64_t to,
                                         Index index) {
    for (int64_t q = from; q < to; q += kBatch) {
        int64_t r[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) r[u] = index(q + u < to ? q + u : to - 1);
        Pack<typename E::S, N> x[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            x[u] = *reinterpret_cast<const Pack<typename E::S, N>*>(rows + r[u] * dim + col);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            for (int k = 0; k < N; ++k) {
                const float y = E::load(x[u].v[k]);
                acc[k] += q + u < to ? y : 0.f;
            }
    }
}

// Keeps a loaded pack's load where it stands.
template <typename S, int N>
__device__ __forceinline__ void pin(Pack<S, N>& p) {
    if constexpr (sizeof(S) * N == 4) {
        uint32_t w = __builtin_bit_cast(uint32_t, p);
        asm volatile("" : "+v"(w));
        p = __builtin_bit_cast(Pack<S, N>, w);
    } else if constexpr (sizeof(S) * N > 4) {
        typedef uint32_t Words __attribute__((ext_vector_type(sizeof(S) * N / 4)));
        Words w = __builtin_bit_cast(Words, p);
        asm volatile("" : "+v"(w));
        p = __builtin_bit_cast(Pack<S, N>, w);
    } else {
        asm volatile("" : "+v"(p.v[0]));
    }
}

// The sums of one call: where the parts of runs that cross tiles go.
struct Parts {
    float* first;  // [tiles, dim] the part of a run that enters the tile, or fills it
    float* last;   // [tiles, dim] the part of a run that leaves it, where it did not enter it
};

// A group of lanes adds up the kSpan places of a tile, kBatch rows in flight
// whatever runs they belong to, and stores a run that lies in the tile as the
// row it is; parts of others go to `parts`.  So the gather is spread evenly
// however often a node occurs.  Marks the runs by output row: the node, or
// (ranks given) its rank among the nodes.
template <typename E, typename O, int N>
__global__ __launch_bounds__(kBlock) void span_sum_kernel(
    const typename E::S* __restrict__ rows, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ places, const uint32_t* __restrict__ valid,
    const uint32_t* __restrict__ ranks, RowShape shape, float scale, Parts parts,
    uint2* __restrict__ runs, typename O::S* __restrict__ out) {
    const int lane = threadIdx.x & ((1 << shape.lanes_log) - 1);
    const int32_t col = ((blockIdx.y << shape.lanes_log) + lane) * N;
    if (col >= shape.dim) return;
    const int64_t groups = static_cast<int64_t>(gridDim.x) * (kBlock >> shape.lanes_log);
    const bool marks = lane == 0 && blockIdx.y == 0;
    const int64_t n = *valid;
    for (int64_t p = (blockIdx.x * static_cast<int64_t>(kBlock) + threadIdx.x) >> shape.lanes_log;
         p * kSpan < n; p += groups) {
        const int64_t begin = p * kSpan;
        const int64_t end = begin + kSpan < n ? begin + kSpan : n;
        uint32_t node = keys[begin];
        const bool enters = begin > 0 && keys[begin - 1] == node;
        int64_t rank = ranks ? static_cast<int64_t>(ranks[p]) - enters : 0;
        if (marks && !enters) runs[ranks ? rank : node].x = static_cast<uint32_t>(begin);
        bool first = true;  // no run has ended in the tile yet
        float acc[N] = {};
        for (int64_t i = begin; i < end; i += kBatch) {
            uint32_t key[kBatch];
            Pack<typename E::S, N> x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int64_t at = i + u < end ? i + u : end - 1;
                key[u] = keys[at];
                x[u] = *reinterpret_cast<const Pack<typename E::S, N>*>(
                    rows + static_cast<int64_t>(places[at]) * shape.dim + col);
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) pin(x[u]);
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (key[u] != node) {
                    const int64_t row = ranks ? rank : static_cast<int64_t>(node);
                    if (first && enters) {
                        store_pack<F32, N>(parts.first + p * shape.dim + col, acc);
                    } else {
#pragma unroll
                        for (int k = 0; k < N; ++k) acc[k] *= scale;
                        store_pack<O, N>(out + row * shape.dim + col, acc);
                    }
                    if (marks) {
                        runs[row].y = static_cast<uint32_t>(i + u);
                        runs[ranks ? rank + 1 : static_cast<int64_t>(key[u])].x =
                            static_cast<uint32_t>(i + u);
                    }
                    first = false;
                    node = key[u];
                    ++rank;
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const float y = E::load(x[u].v[k]);
                    acc[k] += i + u < end ? y : 0.f;
                }
            }
        }
        const bool leaves = end < n && keys[end] == node;
        const int64_t row = ranks ? rank : static_cast<int64_t>(node);
        if (first && enters) {
            store_pack<F32, N>(parts.first + p * shape.dim + col, acc);
        } else if (leaves) {
            store_pack<F32, N>((first ? parts.first : parts.last) + p * shape.dim + col, acc);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] *= scale;
            store_pack<O, N>(out + row * shape.dim + col, acc);
        }
        if (marks && !leaves) runs[row].y = static_cast<uint32_t>(end);
    }
}

// sums[p, :] <- the sum of kFan entries of the level below, for the tiles of
// `span` places that lie in one run.
template <int N>
__global__ __launch_bounds__(kBlock) void tile_sum_kernel(const uint32_t* __restrict__ keys,
                                                          const uint32_t* __restrict__ valid,
                                                          int64_t span,
                                                          const float* __restrict__ below,
                                                          RowShape shape,
                                                          float* __restrict__ sums) {
    const int lane = threadIdx.x & ((1 << shape.lanes_log) - 1);
    const int32_t col = ((blockIdx.y << shape.lanes_log) + lane) * N;
    const int64_t p =
        (blockIdx.x * static_cast<int64_t>(kBlock) + threadIdx.x) >> shape.lanes_log;
    if ((p + 1) * span > *valid || keys[p * span] != keys[(p + 1) * span - 1] || col >= shape.dim)
        return;
    float acc[N] = {};
    add_rows<F32, N>(acc, below, shape.dim, col, p * kFan, (p + 1) * kFan,
                     [](int64_t q) { return q; });
    store_pack<F32, N>(sums + p * shape.dim + col, acc);
}

struct TileSums {
    const float* p[kMaxLevels];
    int32_t levels;
};

// Puts the runs that cross tiles together, each by the group of the tile in
// which it starts: neighbouring nodes, and those a power of two apart, are often
// hubs together, and a group a row would add up one hub after the other.
template <typename O, int N>
__global__ __launch_bounds__(kBlock) void run_sum_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ valid,
    const uint32_t* __restrict__ ranks, const uint2* __restrict__ runs, Parts parts, TileSums tiles,
    RowShape shape, float scale, typename O::S* __restrict__ out) {
    const int lane = threadIdx.x & ((1 << shape.lanes_log) - 1);
    const int64_t per = kBlock >> shape.lanes_log;  // groups a block
    const int64_t own = threadIdx.x >> shape.lanes_log;
    const int32_t col = ((blockIdx.y << shape.lanes_log) + lane) * N;
    if (col >= shape.dim) return;
    const int64_t n = *valid;
    for (int64_t p = blockIdx.x * per + own; (p + 1) * kSpan < n; p += gridDim.x * per) {
        const uint32_t node = keys[(p + 1) * kSpan - 1];
        const bool leaves = keys[(p + 1) * kSpan] == node;
        const bool entered = p > 0 && keys[p * kSpan - 1] == node;
        if (!leaves || entered) continue;
        const int64_t row = ranks ? static_cast<int64_t>(ranks[p + 1]) - 1 : node;
        const uint2 run = runs[row];
        float acc[N] = {};
        int64_t lo = p, hi = (run.y - 1) / kSpan + 1;  // the run's tiles
        if (run.x % kSpan) {  // it starts inside its first tile
            load_pack<F32, N>(acc, parts.last + lo * shape.dim + col);
            ++lo;
        }
        // the parts before the first whole tile of tiles and after the last
        // one, then the same a level up; parts from `full` on are not whole
        int64_t full = run.y / kSpan;
        for (int level = 0;; ++level) {
            const int64_t first = (lo + kFan - 1) / kFan, last = full / kFan;
            const bool more = level < tiles.levels && first < last;
            const int64_t head = more ? first * kFan - lo : hi - lo;
            const int64_t tail = more ? last * kFan - head : 0;  // of entry head on
            const int64_t count = more ? head + hi - last * kFan : head;
            add_rows<F32, N>(acc, level == 0 ? parts.first : tiles.p[level - 1], shape.dim, col, 0,
                             count, [&](int64_t q) { return q < head ? lo + q : tail + q; });
            if (!more) break;
            lo = first;
            hi = full = last;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] *= scale;
        store_pack<O, N>(out + row * shape.dim + col, acc);
    }
}

// ------------------------------------------------------------- few places

// The whole gradient of up to kSmallPlaces places in one launch: a block takes
// the nodes [block * per, ...) of the table.  It writes their zeros, picks their
// places out of the whole list, in order, sorts them by node in LDS, and its
// groups of lanes add up equal shares of them; a run that crosses shares is put
// together from the parts that the groups left in LDS.
//
// Bound by latencies: 12,000 rows of 64 float32 into 2,708 take 16 us; sorted by
// one block and added up by two more launches 38.
template <typename E, typename O, int N>
__global__ __launch_bounds__(kSmallThreads) void few_sum_kernel(
    const typename E::S* __restrict__ rows, Nodes nodes, int32_t count, int64_t per, int bits,
    int passes, RowShape shape, float scale, typename O::S* __restrict__ out,
    int64_t* __restrict__ work) {
    static_assert(N <= 4, "the parts fit LDS");
    __shared__ SmallSort l;
    __shared__ __align__(16) float parts[kSmallThreads][N];  // of the run that enters a share
    const int t = threadIdx.x, w = t / kWave, lane = t & ((1 << shape.lanes_log) - 1);
    const int group = t >> shape.lanes_log, groups = kSmallThreads >> shape.lanes_log;
    const int32_t col = ((blockIdx.y << shape.lanes_log) + lane) * N;
    const bool active = col < shape.dim;
    const int64_t lo = blockIdx.x * per;
    const int64_t hi = lo + per < nodes.num_rows ? lo + per : nodes.num_rows;
    bool bad = false;
    int items = (count + kSmallThreads - 1) / kSmallThreads;
    const int32_t base = w * items * kWave + t % kWave;
    int32_t v[kItems];
    load_nodes(v, nodes, base, kWave, count, bad);
    const float zeros[N] = {};
    if (active)
        for (int64_t r = lo + group; r < hi; r += groups)
            store_pack<O, N>(out + r * shape.dim + col, zeros);
    // the block's places, in order (wavefront, slot, lane)
    uint64_t own[kItems];
    uint32_t in_wave = 0;
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        own[s] = __ballot(s < items && v[s] >= lo && v[s] < hi);
        in_wave += __popcll(own[s]);
    }
    if (t % kWave == 0) l.tot[w] = in_wave;
    const int any_bad = __syncthreads_or(bad);
    if (blockIdx.x == 0 && blockIdx.y == 0 && t < MLXC_WORK_WORDS)
        work[t] = t == 0 && any_bad ? MLXC_STATUS_BAD_NODE : 0;
    uint32_t at = 0;
    int32_t n = 0;
#pragma unroll
    for (int k = 0; k < kSmallWaves; ++k) {
        at += k < w ? l.tot[k] : 0;
        n += l.tot[k];
    }
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        if ((own[s] >> (t % kWave)) & 1) {
            const uint32_t j = at + lane_rank(own[s]);
            l.keys[j] = static_cast<uint32_t>(v[s] - lo);
            l.places[j] = static_cast<uint16_t>(base + s * kWave);
        }
        at += __popcll(own[s]);
    }
    __syncthreads();
    if (n == 0) return;
    for (int pass = 0; pass < passes; ++pass) {
        uint32_t key[kItems], place[kItems];
        const uint32_t have = small_entries(l, key, place, n, items);
        small_pass(l, key, place, have, items, pass * bits, bits, n);
    }
    // equal shares, whole batches while there are few
    const int32_t share = (n + groups - 1) / groups > kBatch ? (n + groups - 1) / groups : kBatch;
    const int32_t begin = group * share < n ? group * share : n;
    const int32_t end = n - begin < share ? n : begin + share;
    uint32_t node = begin < n ? l.keys[begin] : 0;
    const bool enters = begin > 0 && begin < n && l.keys[begin - 1] == node;
    bool first = true;  // no run has ended in the share yet
    float acc[N] = {};
    for (int32_t i = begin; i < end; i += kBatch) {
        Pack<typename E::S, N> x[kBatch];
        uint32_t key[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int32_t q = i + u < end ? i + u : end - 1;
            key[u] = l.keys[q];
            x[u] = *reinterpret_cast<const Pack<typename E::S, N>*>(
                rows + static_cast<int64_t>(l.places[q]) * shape.dim + (active ? col : 0));
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) pin(x[u]);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (key[u] != node) {
                if (first && enters) {
                    store_pack<F32, N>(parts[t], acc);
                } else if (active) {
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] *= scale;
                    store_pack<O, N>(out + (lo + node) * shape.dim + col, acc);
                }
                first = false;
                node = key[u];
#pragma unroll
                for (int k = 0; k < N; ++k) acc[k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const float y = E::load(x[u].v[k]);
                acc[k] += i + u < end ? y : 0.f;
            }
        }
    }
    const bool leaves = begin < n && end < n && l.keys[end] == node;
    if (first && enters) store_pack<F32, N>(parts[t], acc);
    __syncthreads();
    if (begin >= n || (first && enters) || !active) return;
    if (leaves) {  // the shares after this one, until the run ends
        int32_t g = group + 1;
        for (bool more = true; more; ++g) {
            float x[N];
            load_pack<F32, N>(x, parts[(g << shape.lanes_log) | lane]);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += x[k];
            const int32_t next = (g + 1) * share;
            more = next < n && l.keys[next] == node;
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] *= scale;
    store_pack<O, N>(out + (lo + node) * shape.dim + col, acc);
}

__global__ void clear_words_kernel(int64_t* words, int n) {
    if (static_cast<int>(threadIdx.x) < n) words[threadIdx.x] = 0;
}

// ------------------------------------------------------------- host side

size_t round256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// Calls that few_sum_kernel takes, which works in LDS.
bool few_places(int64_t num_rows, int64_t count, bool sparse) {
    return !sparse && num_rows > 0 && count > 0 && count <= kSmallPlaces;
}

// The workspace: the header, and for more places the sort's part, then the sums'.
struct GradLayout {
    size_t sort = 0, runs = 0, first = 0, last = 0, sums[kMaxLevels] = {}, bytes = 0;
    int levels = 0;
    bool few = false;
};

GradLayout grad_layout(int64_t num_rows, int32_t dim, int64_t count, bool sparse) {
    GradLayout l;
    size_t at = round256(MLXC_WORK_WORDS * sizeof(int64_t));
    l.few = few_places(num_rows, count, sparse);
    if (l.few) {
        l.bytes = at;
        return l;
    }
    auto take = [&at](size_t bytes) {
        const size_t a = at;
        at += round256(bytes);
        return a;
    };
    l.sort = take(place_sort_bytes(num_rows, count, sparse));
    const int64_t num_out = sparse && count < num_rows ? count : num_rows;
    const int64_t spans = (count + kSpan - 1) / kSpan;
    l.runs = take(static_cast<size_t>(num_out) * sizeof(uint2));
    l.first = take(static_cast<size_t>(spans) * dim * 4);
    l.last = take(static_cast<size_t>(spans) * dim * 4);
    for (int64_t span = kSpan * kFan; l.levels < kMaxLevels && count / span >= kLevelTiles;
         span *= kFan)
        l.sums[l.levels++] = take(static_cast<size_t>(count / span) * dim * 4);
    l.bytes = at;
    return l;
}

template <typename T>
T* at(void* p, size_t offset) {
    return reinterpret_cast<T*>(static_cast<unsigned char*>(p) + offset);
}

RowShape row_shape(int32_t dim, int n) {
    RowShape s{dim, 0};
    while (s.lanes_log < 6 && (n << s.lanes_log) < dim) ++s.lanes_log;
    return s;
}

// Blocks for `rows` rows of this shape (fewer where a launch would hold 2^32
// threads: the kernels go on by the grid's groups), and the columns' share of
// the grid.
dim3 row_grid(int64_t rows, const RowShape& s, int n) {
    const int64_t per = kBlock >> s.lanes_log;
    int64_t blocks = (rows + per - 1) / per;
    if (blocks > (1 << 23)) blocks = 1 << 23;
    const int32_t cols = n << s.lanes_log;
    return dim3(static_cast<unsigned>(blocks < 1 ? 1 : blocks), (s.dim + cols - 1) / cols);
}

template <typename E, int N>
int embedding_typed(const Table& table, const Nodes& nodes, int64_t count, float scale, void* out,
                    int64_t* status, hipStream_t stream) {
    const uint32_t packs = table.dim / N;
    const uint32_t inverse = packs > 1 ? 0xffffffffu / packs + 1 : 0;
    const bool streamed = static_cast<size_t>(count) * table.dim * sizeof(typename E::S) >
                          (size_t{128} << 20);
    // (1 M rows of 100 bfloat16, two pieces of 8 bytes: 80 us by pieces, 85 whole; of
    // 50 float32 114 and 85)
    constexpr int all = 16 / sizeof(typename E::S);
    if constexpr (N < all && (all / N >= 4 || sizeof(typename E::S) == 4)) {
        if (table.dim >= all && table.num_rows > 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
            int64_t grid = (count * table.dim + kBlock * all - 1) / (kBlock * all);
            if (grid > (int64_t{1} << 22)) grid = int64_t{1} << 22;
            auto* odd = streamed ? embedding_odd_kernel<E, N, true> : embedding_odd_kernel<E, N, false>;
            hipLaunchKernelGGL(odd, dim3(grid), dim3(kBlock), 0, stream,
                               static_cast<const typename E::S*>(table.p), table.row_stride,
                               static_cast<uint32_t>(table.dim), 0xffffffffu / table.dim + 1, nodes,
                               count, scale, static_cast<typename E::S*>(out), status);
            MLXC_HIP_TRY(hipGetLastError());
            return MLXC_OK;
        }
    }
    const int64_t chunk = kBlock * (streamed ? 4 : 1);
    int64_t blocks = (count * packs + chunk - 1) / chunk;
    if (blocks > (int64_t{1} << 22)) blocks = int64_t{1} << 22;
    auto* kernel = streamed ? embedding_kernel<E, N, 4, true> : embedding_kernel<E, N, 1, false>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kBlock), 0, stream,
                       static_cast<const typename E::S*>(table.p), table.row_stride, packs,
                       inverse, nodes, count, scale, static_cast<typename E::S*>(out), status);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

// The sums' buffers, shared by the kernels that fill and read them.
struct SumCall {
    SortedPlaces sorted;
    Nodes nodes;
    const void* rows;
    int32_t dim;
    int64_t count;
    float scale;
    const GradLayout& l;
    void* ws;
    GradOut out;
};

template <typename E, typename O, int N>
int few_launch(const SumCall& c, const RowShape& shape, hipStream_t stream) {
    DeviceInfo info;
    if (int rc = device_info(info)) return rc;
    const int64_t per = (c.nodes.num_rows + info.cus - 1) / info.cus;
    const int all = bits_below(per);
    const int passes = (all + kDigitBits - 1) / kDigitBits;
    const int bits = passes > 0 ? (all + passes - 1) / passes : 1;
    const int32_t cols = N << shape.lanes_log;
    hipLaunchKernelGGL((few_sum_kernel<E, O, N>),
                       dim3(static_cast<unsigned>((c.nodes.num_rows + per - 1) / per),
                            (shape.dim + cols - 1) / cols),
                       dim3(kSmallThreads), 0, stream, static_cast<const typename E::S*>(c.rows),
                       c.nodes, static_cast<int32_t>(c.count), per, bits, passes, shape, c.scale,
                       static_cast<typename O::S*>(c.out.p), static_cast<int64_t*>(c.ws));
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E, typename O, int N>
int sums_typed(const SumCall& c, hipStream_t stream) {
    const RowShape shape = row_shape(c.dim, N);
    if (c.l.few) {
        if constexpr (N <= 4) return few_launch<E, O, N>(c, shape, stream);
    }
    const SortedPlaces& p = c.sorted;
    const Parts parts{at<float>(c.ws, c.l.first), at<float>(c.ws, c.l.last)};
    uint2* runs = at<uint2>(c.ws, c.l.runs);
    typename O::S* out = static_cast<typename O::S*>(c.out.p);
    hipLaunchKernelGGL((span_sum_kernel<E, O, N>),
                       row_grid((c.count + kSpan - 1) / kSpan, shape, N), dim3(kBlock), 0, stream,
                       static_cast<const typename E::S*>(c.rows), p.keys, p.places, p.valid, p.ranks,
                       shape, c.scale, parts, runs, out);
    MLXC_HIP_TRY(hipGetLastError());
    if (c.count <= kSpan) return MLXC_OK;  // one tile
    TileSums tiles{};
    int64_t span = kSpan;
    for (int k = 0; k < c.l.levels; ++k) {
        span *= kFan;
        float* sums = at<float>(c.ws, c.l.sums[k]);
        hipLaunchKernelGGL((tile_sum_kernel<N>), row_grid(c.count / span, shape, N), dim3(kBlock), 0,
                           stream, p.keys, p.valid, span, k == 0 ? parts.first : tiles.p[k - 1],
                           shape, sums);
        MLXC_HIP_TRY(hipGetLastError());
        tiles.p[k] = sums;
        tiles.levels = k + 1;
    }
    hipLaunchKernelGGL((run_sum_kernel<O, N>), row_grid(c.count / kSpan, shape, N), dim3(kBlock), 0,
                       stream, p.keys, p.valid, p.ranks, runs, parts, tiles, shape, c.scale, out);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E, typename O>
int sums_packed(const SumCall& c, hipStream_t stream) {
    // a pack of up to 16 bytes of the rows; its sums and results are stored in
    // one or two instructions, which the same alignment serves
    constexpr int most = 16 / sizeof(typename E::S);
    const int n = pack_width(c.rows, c.dim, c.dim, sizeof(typename E::S), most);
    const int m = pack_width(c.out.p, c.dim, c.dim, sizeof(typename O::S), n);
    if constexpr (most == 8 && sizeof(typename O::S) == 2)  // (eight float32 are two packs)
        if (m >= 8 && !c.l.few) return sums_typed<E, O, most>(c, stream);
    if (m >= 4) return sums_typed<E, O, 4>(c, stream);
    if (m >= 2) return sums_typed<E, O, 2>(c, stream);
    return sums_typed<E, O, 1>(c, stream);
}

template <typename E>
int sums_from(const SumCall& c, hipStream_t stream) {
    if (c.out.dtype == MLXC_FLOAT32) return sums_packed<E, F32>(c, stream);
    if (c.out.dtype == MLXC_BFLOAT16) return sums_packed<E, BF16>(c, stream);
    return sums_packed<E, F16>(c, stream);
}

}  // namespace

int launch_embedding(const Table& table, const Nodes& nodes, int64_t count, float scale, void* out,
                     int64_t* status, hipStream_t stream) {
    if (status) {
        hipLaunchKernelGGL(clear_words_kernel, dim3(1), dim3(kWave), 0, stream, status, 1);
        MLXC_HIP_TRY(hipGetLastError());
    }
    if (count == 0) return MLXC_OK;
    const size_t esz = elem_bytes(table.dtype);
    int n = pack_width(table.p, table.dim, table.row_stride, esz, static_cast<int>(16 / esz));
    n = pack_width(out, table.dim, table.dim, esz, n);
#define MLXC_LOOKUP(E, N) return embedding_typed<E, N>(table, nodes, count, scale, out, status, stream)
    if (table.dtype == MLXC_FLOAT32) {
        if (n == 4) MLXC_LOOKUP(F32, 4);
        if (n == 2) MLXC_LOOKUP(F32, 2);
        MLXC_LOOKUP(F32, 1);
    }
    if (table.dtype == MLXC_BFLOAT16) {
        if (n == 8) MLXC_LOOKUP(BF16, 8);
        if (n == 4) MLXC_LOOKUP(BF16, 4);
        if (n == 2) MLXC_LOOKUP(BF16, 2);
        MLXC_LOOKUP(BF16, 1);
    }
    if (n == 8) MLXC_LOOKUP(F16, 8);
    if (n == 4) MLXC_LOOKUP(F16, 4);
    if (n == 2) MLXC_LOOKUP(F16, 2);
    MLXC_LOOKUP(F16, 1);
#undef MLXC_LOOKUP
}

size_t grad_workspace_bytes(int64_t num_rows, int32_t dim, int64_t count, bool sparse) {
    return grad_layout(num_rows, dim, count, sparse).bytes;
}

int launch_embedding_grad(const void* rows, int32_t dtype, int32_t dim, const Nodes& nodes,
                          int64_t count, float scale, const GradOut& out, void* workspace,
                          hipStream_t stream) {
    const bool sparse = out.ids != nullptr;
    const GradLayout l = grad_layout(nodes.num_rows, dim, count, sparse);
    const int64_t num_out =
        sparse ? (count < nodes.num_rows ? count : nodes.num_rows) : nodes.num_rows;
    SumCall c{SortedPlaces{}, nodes, rows, dim, count, scale, l, workspace, out};
    if (!l.few) {
        // zeros everywhere first, beside the sort: rows that no place belongs to
        // keep them
        const size_t bytes = static_cast<size_t>(num_out) * dim * elem_bytes(out.dtype);
        const ClearOut clear{out.p, bytes, bytes > (size_t{128} << 20), out.ids,
                             sparse ? num_out : 0};
        if (int rc = launch_place_sort(nodes, count, clear, static_cast<int64_t*>(workspace),
                                       at<unsigned char>(workspace, l.sort), c.sorted, stream))
            return rc;
        if (count == 0 || num_out == 0) return MLXC_OK;
    }
    if (dtype == MLXC_FLOAT32) return sums_from<F32>(c, stream);
    if (dtype == MLXC_BFLOAT16) return sums_from<BF16>(c, stream);
    return sums_from<F16>(c, stream);
}

}  // namespace mlxc
