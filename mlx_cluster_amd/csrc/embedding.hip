// Embedding lookup with scaling, and its gradient by sorted nodes: the rows of
// a walk's nodes, and their way back.
//
//   lookup     y[i, :] = s * W[x_i, :]
//   gradient   G[v, :] = s * sum over i with x_i = v of g[i, :]
//
// The gradient sorts (node, place) by node, stable, with an LSD radix sort of
// the bits that a node can have, so that a node's places stand together in
// ascending order; then every row adds its places up.  Places without a node
// are dropped by the first pass.  Walks visit hubs tens of thousands of times:
// the sorted places are cut into tiles of 64, tiles of 64 tiles and so on, a
// tile that lies in one node's run is added up once by the tile kernels, and
// the row takes its sum instead of its places.  So no lane adds more than a few
// hundred rows, nothing is added with atomics, and the order of a sum depends
// on the places alone.
#include "train_host.h"

namespace mlxc {

namespace {

// ------------------------------------------------------------- lookup

// One pack of N elements a thread and step; the packs of a row lie on
// consecutive threads.
template <typename E, int N>
__global__ __launch_bounds__(kBlock) void embedding_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, int32_t packs, Nodes nodes,
    int64_t count, float scale, typename E::S* __restrict__ out, int64_t* status) {
    const int64_t total = count * packs;
    bool bad = false;
    for (int64_t e = blockIdx.x * static_cast<int64_t>(kBlock) + threadIdx.x; e < total;
         e += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t i = e / packs;
        const int64_t d = (e - i * packs) * N;
        const int64_t v = node_at(nodes, i, bad);
        float x[N];
        if (v >= 0) {
            load_pack<E, N>(x, weight + v * row_stride + d);
#pragma unroll
            for (int q = 0; q < N; ++q) x[q] *= scale;
        } else {
#pragma unroll
            for (int q = 0; q < N; ++q) x[q] = 0.f;
        }
        store_pack<E, N>(out + e * N, x);
    }
    report_bad(bad, status);
}

// ------------------------------------------------------------- sort by node

constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kItems = 16;               // keys a thread
constexpr int kTile = kBlock * kItems;   // keys a block
constexpr int kWaves = kBlock / kWave;
constexpr int kWaveTile = kWave * kItems;
static_assert(kDigits == kBlock, "one digit a thread");

// Words of the workspace header.
constexpr int kWordStatus = 0;
constexpr int kWordDistinct = 1;  // distinct nodes (coalesced)

// Exclusive prefix of one value a thread over the block; *total the sum.  `tot`
// is kWaves words of LDS.  Contains two barriers.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* tot, uint32_t* total) {
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t u = __shfl_up(inc, o, kWave);
        if (lane >= o) inc += u;
    }
    if (lane == kWave - 1) tot[w] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int k = 0; k < kWaves; ++k) {
        if (k < w) before += tot[k];
        all += tot[k];
    }
    *total = all;
    __syncthreads();
    return before + inc - v;
}

// Lanes of the wavefront that are active and hold this lane's digit.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool active) {
    uint64_t peers = __ballot(active);
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
        const bool bit = (d >> b) & 1;
        const uint64_t set = __ballot(bit);
        peers &= bit ? set : ~set;
    }
    return peers;
}

// The keys of a pass: the call's nodes (places are their indices, count of
// them), or the last pass's, *valid of them.
struct SortIn {
    Nodes nodes;
    int64_t count;
    const uint32_t* keys;
    const uint32_t* places;
    const uint32_t* valid;
};

// counts[d * tiles + tile] <- the tile's keys of digit d.  The first pass also
// checks the nodes, and zeroes the words that later kernels need zeroed.
template <bool kFirst>
__global__ __launch_bounds__(kBlock) void digit_count_kernel(SortIn in, int shift, uint32_t tiles,
                                                             uint32_t* __restrict__ counts,
                                                             uint32_t* __restrict__ zero,
                                                             int64_t zero_words,
                                                             int64_t* __restrict__ work) {
    __shared__ uint32_t cnt[kDigits];
    const int t = threadIdx.x;
    cnt[t] = 0;
    __syncthreads();
    const int64_t n = kFirst ? in.count : static_cast<int64_t>(*in.valid);
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
    bool bad = false;
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        const int64_t i = base + s * kBlock + t;
        if (i >= n) break;
        const int64_t key = kFirst ? node_at(in.nodes, i, bad) : static_cast<int64_t>(in.keys[i]);
        if (key >= 0) atomicAdd(&cnt[(static_cast<uint32_t>(key) >> shift) & (kDigits - 1)], 1u);
    }
    __syncthreads();
    counts[static_cast<size_t>(t) * tiles + blockIdx.x] = cnt[t];
    if (kFirst) {
        for (int64_t k = blockIdx.x * static_cast<int64_t>(kBlock) + t; k < zero_words;
             k += static_cast<int64_t>(gridDim.x) * kBlock)
            zero[k] = 0;
        report_bad(bad, work + kWordStatus);
    }
}

// Exclusive prefix over each digit's tiles, in place, one block a digit;
// totals[digit] <- the sum.
__global__ __launch_bounds__(kBlock) void digit_prefix_kernel(uint32_t* __restrict__ counts,
                                                              uint32_t tiles,
                                                              uint32_t* __restrict__ totals) {
    __shared__ uint32_t tot[kWaves];
    uint32_t* row = counts + static_cast<size_t>(blockIdx.x) * tiles;
    uint32_t carry = 0;
    for (uint32_t base = 0; base < tiles; base += kBlock) {
        const uint32_t j = base + threadIdx.x;
        const uint32_t v = j < tiles ? row[j] : 0;
        uint32_t all;
        const uint32_t ex = block_prefix(v, tot, &all);
        if (j < tiles) row[j] = carry + ex;
        carry += all;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Stable: a key's output place is the keys of lower digits, those of its digit
// in earlier tiles, and those before it in its tile (wavefront, slot, lane).
template <bool kFirst>
__global__ __launch_bounds__(kBlock) void digit_scatter_kernel(
    SortIn in, int shift, uint32_t tiles, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, uint32_t* __restrict__ keys_out,
    uint32_t* __restrict__ places_out, uint32_t* __restrict__ valid_out) {
    __shared__ uint32_t cnt[kWaves][kDigits];
    __shared__ uint32_t tot[kWaves];
    const int t = threadIdx.x, w = t / kWave, lane = t % kWave;
    for (int k = 0; k < kWaves; ++k) cnt[k][t] = 0;
    uint32_t all;
    const uint32_t digit_base = block_prefix(totals[t], tot, &all);
    if (kFirst && blockIdx.x == 0 && t == 0) *valid_out = all;
    const uint32_t tile_base = counts[static_cast<size_t>(t) * tiles + blockIdx.x];
    const int64_t n = kFirst ? in.count : static_cast<int64_t>(*in.valid);
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile + w * kWaveTile + lane;
    uint32_t key[kItems], place[kItems], rank[kItems];
    uint32_t have = 0;
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        const int64_t i = base + s * kWave;
        bool ok = i < n;
        key[s] = place[s] = 0;
        if (ok) {
            if (kFirst) {
                bool bad = false;
                const int64_t v = node_at(in.nodes, i, bad);
                ok = v >= 0;
                key[s] = static_cast<uint32_t>(v);
                place[s] = static_cast<uint32_t>(i);
            } else {
                key[s] = in.keys[i];
                place[s] = in.places[i];
            }
        }
        have |= static_cast<uint32_t>(ok) << s;
    }
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        const bool ok = (have >> s) & 1;
        const uint32_t d = (key[s] >> shift) & (kDigits - 1);
        const uint64_t peers = same_digit(d, ok);
        const uint32_t before = cnt[w][d];
        const int r = lane_rank(peers);
        rank[s] = before + r;
        // the first of the peers writes after all of them have read (one
        // wavefront: in order)
        if (ok && r == 0) cnt[w][d] = before + __popcll(peers);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    uint32_t at = digit_base + tile_base;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        const uint32_t c = cnt[k][t];
        cnt[k][t] = at;
        at += c;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        if (!((have >> s) & 1)) continue;
        const uint32_t to = cnt[w][(key[s] >> shift) & (kDigits - 1)] + rank[s];
        keys_out[to] = key[s];
        places_out[to] = place[s];
    }
}

// ------------------------------------------------------------- runs

// Dense: the run of every node that occurs, [runs[v].x, runs[v].y) of the
// sorted places; runs is zeroed before.
__global__ __launch_bounds__(kBlock) void mark_runs_kernel(const uint32_t* __restrict__ keys,
                                                           const uint32_t* __restrict__ valid,
                                                           uint2* __restrict__ runs) {
    const int64_t n = *valid;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kBlock) + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * kBlock) {
        const uint32_t k = keys[i];
        if (i == 0 || keys[i - 1] != k) runs[k].x = static_cast<uint32_t>(i);
        if (i == n - 1 || keys[i + 1] != k) runs[k].y = static_cast<uint32_t>(i + 1);
    }
}

// Coalesced: heads[chunk] <- the runs that start in a chunk of kTile places.
__global__ __launch_bounds__(kBlock) void count_heads_kernel(const uint32_t* __restrict__ keys,
                                                             const uint32_t* __restrict__ valid,
                                                             uint32_t* __restrict__ heads) {
    __shared__ uint32_t tot[kWaves];
    const int64_t n = *valid, base = static_cast<int64_t>(blockIdx.x) * kTile;
    uint32_t c = 0;
    for (int s = 0; s < kItems; ++s) {
        const int64_t i = base + s * kBlock + threadIdx.x;
        c += i < n && (i == 0 || keys[i - 1] != keys[i]);
    }
    uint32_t all;
    block_prefix(c, tot, &all);
    if (threadIdx.x == 0) heads[blockIdx.x] = all;
}

// ... and run u's start, its node, and the number of runs.
__global__ __launch_bounds__(kBlock) void list_runs_kernel(const uint32_t* __restrict__ keys,
                                                           const uint32_t* __restrict__ valid,
                                                           const uint32_t* __restrict__ heads,
                                                           uint32_t* __restrict__ starts,
                                                           int64_t* __restrict__ ids,
                                                           int64_t* __restrict__ work) {
    __shared__ uint32_t tot[kWaves];
    const int64_t n = *valid, base = static_cast<int64_t>(blockIdx.x) * kTile;
    uint32_t part = 0, before;
    for (uint32_t k = threadIdx.x; k < blockIdx.x; k += kBlock) part += heads[k];
    block_prefix(part, tot, &before);
    const int64_t first = base + static_cast<int64_t>(threadIdx.x) * kItems;
    uint32_t is_head = 0;
    for (int s = 0; s < kItems; ++s) {
        const int64_t i = first + s;
        if (i < n && (i == 0 || keys[i - 1] != keys[i])) is_head |= 1u << s;
    }
    uint32_t all;
    uint32_t u = before + block_prefix(__popc(is_head), tot, &all);
    for (int s = 0; s < kItems; ++s) {
        if (!((is_head >> s) & 1)) continue;
        starts[u] = static_cast<uint32_t>(first + s);
        ids[u++] = keys[first + s];
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) work[kWordDistinct] = before + all;
}

// ------------------------------------------------------------- sums

// Tile sums: level l's tile p covers the sorted places [p * 64^l, (p + 1) *
// 64^l), for l = 1 .. levels.
constexpr int kFan = 64;
constexpr int kMaxLevels = 3;

// The lanes that serve one row: 2^lanes_log of them, a pack of N columns each,
// from column first_column on.
struct RowShape {
    int32_t dim;
    int32_t lanes_log;
};

template <typename E, int N>
__device__ __forceinline__ void add_row(float (&acc)[N], const typename E::S* row) {
    float x[N];
    load_pack<E, N>(x, row);
#pragma unroll
    for (int q = 0; q < N; ++q) acc[q] += x[q];
}

// sums[p, :] <- the sum of tile p's kFan rows (level 1: the rows of its places,
// E; above: the level below's sums) where the tile lies in one run.
template <typename E, int N, bool kRows>
__global__ __launch_bounds__(kBlock) void tile_sum_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ valid, int64_t span,
    const typename E::S* __restrict__ rows, const uint32_t* __restrict__ places, RowShape shape,
    float* __restrict__ sums) {
    const int lane = threadIdx.x & ((1 << shape.lanes_log) - 1);
    const int64_t groups = static_cast<int64_t>(gridDim.x) * (kBlock >> shape.lanes_log);
    const int32_t col = ((blockIdx.y << shape.lanes_log) + lane) * N;
    const int64_t n = *valid;
    for (int64_t p = (blockIdx.x * static_cast<int64_t>(kBlock) + threadIdx.x) >> shape.lanes_log;
         (p + 1) * span <= n; p += groups) {
        if (keys[p * span] != keys[(p + 1) * span - 1] || col >= shape.dim) continue;
        float acc[N] = {};
#pragma unroll 4
        for (int q = 0; q < kFan; ++q) {
            const int64_t r = kRows ? static_cast<int64_t>(places[p * kFan + q]) : p * kFan + q;
            add_row<E, N>(acc, rows + r * shape.dim + col);
        }
        store_pack<F32, N>(sums + p * shape.dim + col, acc);
    }
}

struct TileSums {
    const float* p[kMaxLevels];
    int32_t levels;
};

// Every row of the output: scale * the sum of its run, tiles where they lie in
// it whole.  Dense: row v's run is runs[v]; coalesced: run u is [starts[u],
// starts[u + 1]), and past the last run rows are zeros and ids -1.
template <typename E, typename O, int N>
__global__ __launch_bounds__(kBlock) void row_sum_kernel(
    const typename E::S* __restrict__ rows, const uint32_t* __restrict__ places,
    const uint32_t* __restrict__ valid, const uint2* __restrict__ runs,
    const uint32_t* __restrict__ starts, const int64_t* __restrict__ work, int64_t* __restrict__ ids,
    TileSums tiles, RowShape shape, int64_t num_out, float scale, typename O::S* __restrict__ out) {
    const int lane = threadIdx.x & ((1 << shape.lanes_log) - 1);
    const int64_t groups = static_cast<int64_t>(gridDim.x) * (kBlock >> shape.lanes_log);
    const int32_t col = ((blockIdx.y << shape.lanes_log) + lane) * N;
    const int64_t distinct = ids ? work[kWordDistinct] : 0;
    for (int64_t v = (blockIdx.x * static_cast<int64_t>(kBlock) + threadIdx.x) >> shape.lanes_log;
         v < num_out; v += groups) {
        int64_t i = 0, end = 0;
        if (!ids) {
            const uint2 r = runs[v];
            i = r.x;
            end = r.y;
        } else if (v < distinct) {
            i = starts[v];
            end = v + 1 < distinct ? starts[v + 1] : *valid;
        } else if (lane == 0 && blockIdx.y == 0) {
            ids[v] = -1;
        }
        if (col >= shape.dim) continue;
        float acc[N] = {};
        while (i < end) {
            // the largest tile that starts here and lies in the run
            int64_t span = 1;
            int level = 0;
            while (level < tiles.levels && i % (span * kFan) == 0 && i + span * kFan <= end) {
                span *= kFan;
                ++level;
            }
            if (level == 0)
                add_row<E, N>(acc, rows + static_cast<int64_t>(places[i]) * shape.dim + col);
            else
                add_row<F32, N>(acc, tiles.p[level - 1] + i / span * shape.dim + col);
            i += span;
        }
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] *= scale;
        store_pack<O, N>(out + v * shape.dim + col, acc);
    }
}

__global__ void clear_words_kernel(int64_t* words, int n) {
    if (static_cast<int>(threadIdx.x) < n) words[threadIdx.x] = 0;
}

// ------------------------------------------------------------- host side

size_t round256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

int bits_below(int64_t n) {  // bits of n - 1
    int b = 0;
    for (uint64_t x = n > 1 ? static_cast<uint64_t>(n - 1) : 0; x; x >>= 1) ++b;
    return b;
}

struct GradLayout {
    int passes = 1;
    uint32_t tiles = 0;
    size_t keys[2], places[2], counts, totals, valid, runs, heads, sums[kMaxLevels], bytes;
    int levels = 0;
};

GradLayout grad_layout(int64_t num_rows, int32_t dim, int64_t count, bool sparse) {
    GradLayout l;
    const int bits = bits_below(num_rows);
    l.passes = bits == 0 ? 1 : (bits + kDigitBits - 1) / kDigitBits;
    l.tiles = static_cast<uint32_t>(count > 0 ? (count + kTile - 1) / kTile : 1);
    size_t at = round256(MLXC_WORK_WORDS * sizeof(int64_t));
    auto take = [&at](size_t bytes) {
        const size_t a = at;
        at += round256(bytes);
        return a;
    };
    for (int b = 0; b < 2; ++b) {
        l.keys[b] = take(static_cast<size_t>(count) * 4);
        l.places[b] = take(static_cast<size_t>(count) * 4);
    }
    l.counts = take(static_cast<size_t>(l.tiles) * kDigits * 4);
    l.totals = take(kDigits * 4);
    l.valid = take(8);
    const int64_t cap = count < num_rows ? count : num_rows;
    l.runs = take(static_cast<size_t>(sparse ? cap * 4 : num_rows * 8));
    l.heads = take(static_cast<size_t>(sparse ? l.tiles : 0) * 4);
    for (int64_t span = kFan; l.levels < kMaxLevels && span <= count; span *= kFan)
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

// Blocks for `rows` rows of this shape, and the columns' share of the grid.
dim3 row_grid(int64_t rows, const RowShape& s, int n, int cus) {
    const int64_t per = kBlock >> s.lanes_log;
    int64_t blocks = (rows + per - 1) / per;
    const int64_t most = static_cast<int64_t>(cus) * 64;
    if (blocks > most) blocks = most;
    const int32_t cols = n << s.lanes_log;
    return dim3(static_cast<unsigned>(blocks < 1 ? 1 : blocks), (s.dim + cols - 1) / cols);
}

template <typename E, int N>
int embedding_typed(const Table& table, const Nodes& nodes, int64_t count, float scale, void* out,
                    int64_t* status, hipStream_t stream) {
    const int32_t packs = table.dim / N;
    DeviceInfo info;
    if (int rc = device_info(info)) return rc;
    int64_t blocks = (count * packs + kBlock - 1) / kBlock;
    if (blocks > info.cus * 64) blocks = info.cus * 64;
    hipLaunchKernelGGL((embedding_kernel<E, N>), dim3(blocks), dim3(kBlock), 0, stream,
                       static_cast<const typename E::S*>(table.p), table.row_stride, packs, nodes,
                       count, scale, static_cast<typename E::S*>(out), status);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

// The sums' buffers, shared by the kernels that fill and read them.
struct SumCall {
    const uint32_t *keys, *places, *valid;
    const void* rows;
    int32_t dim;
    int64_t count, num_out;
    float scale;
    const GradLayout& l;
    void* ws;
    GradOut out;
};

template <typename E, typename O, int N>
int sums_typed(const SumCall& c, hipStream_t stream) {
    DeviceInfo info;
    if (int rc = device_info(info)) return rc;
    const RowShape shape = row_shape(c.dim, N);
    TileSums tiles{};
    int64_t span = 1;
    for (int k = 0; k < c.l.levels; ++k) {
        span *= kFan;
        float* sums = at<float>(c.ws, c.l.sums[k]);
        const dim3 grid = row_grid(c.count / span, shape, N, info.cus);
        if (k == 0)
            hipLaunchKernelGGL((tile_sum_kernel<E, N, true>), grid, dim3(kBlock), 0, stream, c.keys,
                               c.valid, span, static_cast<const typename E::S*>(c.rows), c.places,
                               shape, sums);
        else
            hipLaunchKernelGGL((tile_sum_kernel<F32, N, false>), grid, dim3(kBlock), 0, stream,
                               c.keys, c.valid, span, tiles.p[k - 1], nullptr, shape, sums);
        MLXC_HIP_TRY(hipGetLastError());
        tiles.p[k] = sums;
        tiles.levels = k + 1;
    }
    hipLaunchKernelGGL((row_sum_kernel<E, O, N>), row_grid(c.num_out, shape, N, info.cus),
                       dim3(kBlock), 0, stream, static_cast<const typename E::S*>(c.rows), c.places,
                       c.valid, at<const uint2>(c.ws, c.l.runs), at<const uint32_t>(c.ws, c.l.runs),
                       static_cast<const int64_t*>(c.ws), c.out.ids, tiles, shape, c.num_out,
                       c.scale, static_cast<typename O::S*>(c.out.p));
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E, typename O>
int sums_packed(const SumCall& c, hipStream_t stream) {
    constexpr size_t esz = sizeof(typename E::S), osz = sizeof(typename O::S);
    // a pack is at most 16 bytes of either; the tiles' sums follow the packs,
    // their rows aligned as dim says
    constexpr int most = 16 / (esz > osz ? esz : osz);
    const int n = pack_width(c.rows, c.dim, c.dim, esz, most);
    const int m = pack_width(c.out.p, c.dim, c.dim, osz, n < 4 ? n : 4);
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
    int64_t* work = static_cast<int64_t*>(workspace);
    uint32_t* valid = at<uint32_t>(workspace, l.valid);
    hipLaunchKernelGGL(clear_words_kernel, dim3(1), dim3(kWave), 0, stream, work, MLXC_WORK_WORDS);
    hipLaunchKernelGGL(clear_words_kernel, dim3(1), dim3(kWave), 0, stream,
                       at<int64_t>(workspace, l.valid), 1);
    MLXC_HIP_TRY(hipGetLastError());
    const int64_t num_out =
        sparse ? (count < nodes.num_rows ? count : nodes.num_rows) : nodes.num_rows;
    if (num_out == 0) return MLXC_OK;
    uint32_t* counts = at<uint32_t>(workspace, l.counts);
    uint32_t* totals = at<uint32_t>(workspace, l.totals);
    uint32_t* runs = at<uint32_t>(workspace, l.runs);
    const unsigned blocks = l.tiles;
    int cur = 0;
    for (int pass = 0; pass < l.passes; ++pass) {
        const int shift = pass * kDigitBits;
        const SortIn in{nodes, count, at<uint32_t>(workspace, l.keys[cur]),
                        at<uint32_t>(workspace, l.places[cur]), valid};
        const int to = pass == 0 ? 0 : cur ^ 1;
        uint32_t *keys_out = at<uint32_t>(workspace, l.keys[to]),
                 *places_out = at<uint32_t>(workspace, l.places[to]);
        if (pass == 0) {
            hipLaunchKernelGGL(digit_count_kernel<true>, dim3(blocks), dim3(kBlock), 0, stream, in,
                               shift, l.tiles, counts, runs, sparse ? 0 : 2 * nodes.num_rows, work);
        } else {
            hipLaunchKernelGGL(digit_count_kernel<false>, dim3(blocks), dim3(kBlock), 0, stream, in,
                               shift, l.tiles, counts, nullptr, 0, work);
        }
        MLXC_HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(digit_prefix_kernel, dim3(kDigits), dim3(kBlock), 0, stream, counts,
                           l.tiles, totals);
        MLXC_HIP_TRY(hipGetLastError());
        auto* scatter = pass == 0 ? digit_scatter_kernel<true> : digit_scatter_kernel<false>;
        hipLaunchKernelGGL(scatter, dim3(blocks), dim3(kBlock), 0, stream, in, shift, l.tiles,
                           counts, totals, keys_out, places_out, valid);
        MLXC_HIP_TRY(hipGetLastError());
        cur = to;
    }
    const uint32_t* keys = at<uint32_t>(workspace, l.keys[cur]);
    const uint32_t* places = at<uint32_t>(workspace, l.places[cur]);
    if (sparse) {
        uint32_t* heads = at<uint32_t>(workspace, l.heads);
        hipLaunchKernelGGL(count_heads_kernel, dim3(blocks), dim3(kBlock), 0, stream, keys, valid,
                           heads);
        MLXC_HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(list_runs_kernel, dim3(blocks), dim3(kBlock), 0, stream, keys, valid,
                           heads, runs, out.ids, work);
    } else {
        hipLaunchKernelGGL(mark_runs_kernel, dim3(blocks * 4), dim3(kBlock), 0, stream, keys, valid,
                           reinterpret_cast<uint2*>(runs));
    }
    MLXC_HIP_TRY(hipGetLastError());
    const SumCall c{keys, places, valid, rows, dim, count, num_out, scale, l, workspace, out};
    if (dtype == MLXC_FLOAT32) return sums_from<F32>(c, stream);
    if (dtype == MLXC_BFLOAT16) return sums_from<BF16>(c, stream);
    return sums_from<F16>(c, stream);
}

}  // namespace mlxc
