// Places sorted by node: what a gradient needs to add a node's rows up.
//
// A stable LSD radix sort of (node, place) by the bits that a node can have, so
// that a node's places stand together in ascending order.  Places without a
// node are dropped by the first pass.  The launches also write what the gradient
// needs written everywhere (zeros, ids of -1), by blocks of their own.
//
// Up to 16,384 places are sorted by one block in LDS; longer lists in passes of
// up to 8 bits, two launches each: the digits of every tile are counted, 4,096
// places or (in lists of up to 65,536) 1,024, and its keys moved through LDS to their
// places.  A block adds the counts of the tiles before it up itself while there are
// few of them; else a launch in between does.
#include "place_sort.h"

namespace mlxc {

namespace {

static_assert(kDigits == kBlock, "one digit a thread");

// Keys a thread (kPer below), and with them keys a tile: 16, or 4 in lists of so
// few tiles that a block's own time counts (a coalesced gradient of 48,100 rows
// in 2^24 nodes: 83 -> 60 us).
constexpr int kFewItems = 4;

// Tiles up to which a block adds the counts of all tiles itself, from a
// [tile][digit] array (64 reads a thread, under 3 us); with more they are
// [digit][tile] and digit_prefix_kernel adds them up.
constexpr uint32_t kFlatTiles = 64;

// Zeros and -1s by thread `t` of `threads`.
__device__ __forceinline__ void clear_share(const ClearOut& c, size_t t, size_t threads) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    unsigned char* p = static_cast<unsigned char*>(c.p);
    const size_t lead = (16 - reinterpret_cast<uintptr_t>(p) % 16) % 16;
    const size_t head = lead < c.bytes ? lead : c.bytes;
    const size_t packs = (c.bytes - head) / 16, tail = head + packs * 16;
    u32x4* body = reinterpret_cast<u32x4*>(p + head);
    const u32x4 zero = {0u, 0u, 0u, 0u};
    if (c.streamed) {  // more than the caches keep
        for (size_t i = t; i < packs; i += threads) __builtin_nontemporal_store(zero, body + i);
    } else {
        for (size_t i = t; i < packs; i += threads) body[i] = zero;
    }
    if (t < head) p[t] = 0;
    if (t < c.bytes - tail) p[tail + t] = 0;
    for (size_t i = t; i < static_cast<size_t>(c.num_ids); i += threads) c.ids[i] = -1;
}

// ------------------------------------------------------------- short lists

// Block 0 sorts, the others clear.  Every wavefront ranks its stretch of the
// list by ballots, a digit's keys in order; the places go through LDS.  Bound by
// the one compute unit's vector instructions: 12,000 places of 2,708 nodes 22 us.
__global__ __launch_bounds__(kSmallThreads) void sort_small_kernel(
    Nodes nodes, int32_t count, int bits, int passes, ClearOut clear, uint32_t* __restrict__ keys_out,
    uint32_t* __restrict__ places_out, uint32_t* __restrict__ valid_out,
    uint32_t* __restrict__ ranks, int64_t* __restrict__ work) {
    __shared__ SmallSort l;
    const int t = threadIdx.x;
    if (blockIdx.x > 0) {
        clear.num_ids = 0;  // ids are block 0's
        clear_share(clear, (blockIdx.x - 1) * static_cast<size_t>(kSmallThreads) + t,
                    (gridDim.x - 1) * static_cast<size_t>(kSmallThreads));
        return;
    }
    bool bad = false;
    int32_t n = count;
    uint32_t key[kItems], place[kItems];
    for (int pass = 0; pass < passes; ++pass) {
        int items;
        uint32_t have = 0;
        if (pass == 0) {
            items = (n + kSmallThreads - 1) / kSmallThreads;
            const int32_t base = t / kWave * items * kWave + t % kWave;
            int32_t v[kItems];
            load_nodes(v, nodes, base, kWave, n, bad);
#pragma unroll
            for (int s = 0; s < kItems; ++s) {
                have |= static_cast<uint32_t>(s < items && v[s] >= 0) << s;
                key[s] = v[s];
                place[s] = base + s * kWave;
            }
        } else {
            have = small_entries(l, key, place, n, items);
        }
        small_pass(l, key, place, have, items, pass * bits, bits, n);
    }
    const uint32_t* keys = l.keys;
    for (int32_t i = t; i < n; i += kSmallThreads) {
        keys_out[i] = keys[i];
        places_out[i] = l.places[i];
    }
    const int any_bad = __syncthreads_or(bad);
    if (t == 0) {
        *valid_out = n;
        work[0] = any_bad ? MLXC_STATUS_BAD_NODE : 0;
    } else if (t < MLXC_WORK_WORDS) {
        work[t] = 0;
    }
    if (!ranks) return;
    const int32_t per = (n + kSmallThreads - 1) / kSmallThreads, first = t * per;
    uint32_t heads = 0, all;
    for (int32_t i = first; i < first + per && i < n; ++i) heads += i == 0 || keys[i - 1] != keys[i];
    uint32_t u = block_prefix<kSmallThreads>(heads, l.tot, &all);
    for (int32_t i = first; i < first + per && i < n; ++i) {
        if (i % kSpan == 0) ranks[i / kSpan] = u;
        if (i == 0 || keys[i - 1] != keys[i]) clear.ids[u++] = keys[i];
    }
    for (int64_t i = all + t; i < clear.num_ids; i += kSmallThreads) clear.ids[i] = -1;
}

// ------------------------------------------------------------- passes

// The keys of a pass: the call's nodes (places are their indices, count of
// them), or the last pass's, *valid of them.
struct SortIn {
    Nodes nodes;
    int64_t count;
    const uint32_t* keys;
    const uint32_t* places;
    const uint32_t* valid;
    int shift, bits;  // of the pass's digit
};

__device__ __forceinline__ uint32_t digit_of(const SortIn& in, uint32_t key) {
    return (key >> in.shift) & ((1u << in.bits) - 1);
}

// Where a tile's count of a digit stands.
__device__ __forceinline__ size_t count_at(uint32_t digit, uint32_t tile, uint32_t tiles) {
    return tiles <= kFlatTiles ? static_cast<size_t>(tile) * kDigits + digit
                               : static_cast<size_t>(digit) * tiles + tile;
}

// The tiles' digits counted; blocks from `tiles` on clear.  The first pass also
// notes tiles that hold a bad node.
template <bool kFirst, int kPer>
__global__ __launch_bounds__(kBlock) void digit_count_kernel(SortIn in, uint32_t tiles,
                                                             uint32_t* __restrict__ counts,
                                                             uint32_t* __restrict__ bad_tiles,
                                                             ClearOut clear) {
    __shared__ uint32_t cnt[kDigits];
    const int t = threadIdx.x;
    if (blockIdx.x >= tiles) {
        clear_share(clear, (blockIdx.x - tiles) * static_cast<size_t>(kBlock) + t,
                    (gridDim.x - tiles) * static_cast<size_t>(kBlock));
        return;
    }
    cnt[t] = 0;
    __syncthreads();
    const int64_t n = kFirst ? in.count : static_cast<int64_t>(*in.valid);
    const int64_t base = static_cast<int64_t>(blockIdx.x) * (kBlock * kPer);
    bool bad = false;
    int32_t v[kPer];
    if (kFirst) {
        load_nodes(v, in.nodes, base + t, kBlock, n, bad);
    } else {
#pragma unroll
        for (int s = 0; s < kPer; ++s) {
            const int64_t i = base + s * kBlock + t;
            v[s] = static_cast<int32_t>(n > 0 ? in.keys[i < n ? i : n - 1] : 0);
        }
    }
#pragma unroll
    for (int s = 0; s < kPer; ++s)
        if (base + s * kBlock + t < n && v[s] >= 0) atomicAdd(&cnt[digit_of(in, v[s])], 1u);
    const int any_bad = __syncthreads_or(bad);
    counts[count_at(t, blockIdx.x, tiles)] = cnt[t];
    if (kFirst && t == 0) bad_tiles[blockIdx.x] = any_bad;
}

// Exclusive prefix over each digit's tiles, in place, one block a digit;
// totals[digit] <- the sum.
__global__ __launch_bounds__(kBlock) void digit_prefix_kernel(uint32_t* __restrict__ counts,
                                                              uint32_t tiles,
                                                              uint32_t* __restrict__ totals) {
    __shared__ uint32_t tot[kBlock / kWave];
    uint32_t* row = counts + static_cast<size_t>(blockIdx.x) * tiles;
    uint32_t carry = 0;
    for (uint32_t base = 0; base < tiles; base += kBlock) {
        const uint32_t j = base + threadIdx.x;
        const uint32_t v = j < tiles ? row[j] : 0;
        uint32_t all;
        const uint32_t ex = block_prefix<kBlock>(v, tot, &all);
        if (j < tiles) row[j] = carry + ex;
        carry += all;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Stable: a key's output place is the keys of lower digits, those of its digit
// in earlier tiles, and those before it in its tile (wavefront, slot, lane).  A
// tile's keys are put in order in LDS first, so that a digit's go out together
// (stored from where they were ranked, 377,000 and 5.3 M places took 24.5 us a pass
// together, so 20).
template <bool kFirst, int kPer>
__global__ __launch_bounds__(kBlock) void digit_scatter_kernel(
    SortIn in, uint32_t tiles, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, const uint32_t* __restrict__ bad_tiles,
    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ places_out,
    uint32_t* __restrict__ valid_out, int64_t* __restrict__ work, ClearOut clear) {
    constexpr int kWaves = kBlock / kWave;
    __shared__ uint32_t buf_keys[(kBlock * kPer)], buf_places[(kBlock * kPer)];
    __shared__ uint32_t cnt[kWaves][kDigits];
    __shared__ uint32_t shift_to[kDigits];  // from a place in the tile to one in the list
    __shared__ uint32_t tot[kWaves];
    const int t = threadIdx.x, w = t / kWave, lane = t % kWave;
    if (blockIdx.x >= tiles) {
        clear_share(clear, (blockIdx.x - tiles) * static_cast<size_t>(kBlock) + t,
                    (gridDim.x - tiles) * static_cast<size_t>(kBlock));
        return;
    }
    for (int k = 0; k < kWaves; ++k) cnt[k][t] = 0;
    const int64_t n = kFirst ? in.count : static_cast<int64_t>(*in.valid);
    const int64_t base = static_cast<int64_t>(blockIdx.x) * (kBlock * kPer) + w * (kWave * kPer) + lane;
    uint32_t key[kPer], place[kPer], rank[kPer];
    uint32_t have = 0;
    if (kFirst) {
        bool bad = false;  // (the count has noted it)
        int32_t v[kPer];
        load_nodes(v, in.nodes, base, kWave, n, bad);
#pragma unroll
        for (int s = 0; s < kPer; ++s) {
            have |= static_cast<uint32_t>(v[s] >= 0) << s;
            key[s] = v[s];
            place[s] = static_cast<uint32_t>(base + s * kWave);
        }
    } else {
#pragma unroll
        for (int s = 0; s < kPer; ++s) {
            const int64_t i = base + s * kWave;
            const int64_t at = i < n ? i : n - 1;
            have |= static_cast<uint32_t>(i < n) << s;
            key[s] = n > 0 ? in.keys[at] : 0;
            place[s] = n > 0 ? in.places[at] : 0;
        }
    }
    // digit t's keys in all tiles, and in the tiles before this one
    uint32_t total = 0, before = 0;
    if (tiles <= kFlatTiles) {
#pragma unroll 8
        for (uint32_t k = 0; k < tiles; ++k) {
            const uint32_t c = counts[static_cast<size_t>(k) * kDigits + t];
            total += c;
            before += k < blockIdx.x ? c : 0;
        }
    } else {
        total = totals[t];
        before = counts[static_cast<size_t>(t) * tiles + blockIdx.x];
    }
    uint32_t all;
    const uint32_t digit_base = block_prefix<kBlock>(total, tot, &all);
    if (kFirst && blockIdx.x == 0) {
        uint32_t bad = 0;
        for (uint32_t k = t; k < tiles; k += kBlock) bad |= bad_tiles[k];
        const int any_bad = __syncthreads_or(static_cast<int>(bad));
        if (t == 0) {
            *valid_out = all;
            work[0] = any_bad ? MLXC_STATUS_BAD_NODE : 0;
        } else if (t < MLXC_WORK_WORDS) {
            work[t] = 0;
        }
    }
#pragma unroll
    for (int s = 0; s < kPer; ++s)
        rank[s] = take_rank(cnt[w], digit_of(in, key[s]), in.bits, (have >> s) & 1);
    __syncthreads();
    uint32_t c[kWaves], own = 0;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        c[k] = cnt[k][t];
        own += c[k];
    }
    uint32_t in_tile;
    uint32_t at = block_prefix<kBlock>(own, tot, &in_tile);
    shift_to[t] = digit_base + before - at;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        cnt[k][t] = at;
        at += c[k];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kPer; ++s) {
        if (!((have >> s) & 1)) continue;
        const uint32_t j = cnt[w][digit_of(in, key[s])] + rank[s];
        buf_keys[j] = key[s];
        buf_places[j] = place[s];
    }
    __syncthreads();
    for (uint32_t j = t; j < in_tile; j += kBlock) {
        const uint32_t k = buf_keys[j];
        const uint32_t to = shift_to[digit_of(in, k)] + j;
        keys_out[to] = k;
        places_out[to] = buf_places[j];
    }
}

// ------------------------------------------------------------- distinct nodes

// heads[tile] <- the runs of one node that start in a tile of the sorted places.
template <int kPer>
__global__ __launch_bounds__(kBlock) void count_heads_kernel(const uint32_t* __restrict__ keys,
                                                             const uint32_t* __restrict__ valid,
                                                             uint32_t* __restrict__ heads) {
    __shared__ uint32_t tot[kBlock / kWave];
    const int64_t n = *valid, base = static_cast<int64_t>(blockIdx.x) * (kBlock * kPer);
    uint32_t c = 0;
    for (int s = 0; s < kPer; ++s) {
        const int64_t i = base + s * kBlock + threadIdx.x;
        c += i < n && (i == 0 || keys[i - 1] != keys[i]);
    }
    uint32_t all;
    block_prefix<kBlock>(c, tot, &all);
    if (threadIdx.x == 0) heads[blockIdx.x] = all;
}

// ... then the runs' nodes, and ranks[p] <- the runs that start before the kSpan
// places from p * kSpan on.
template <int kPer>
__global__ __launch_bounds__(kBlock) void list_runs_kernel(const uint32_t* __restrict__ keys,
                                                           const uint32_t* __restrict__ valid,
                                                           const uint32_t* __restrict__ heads,
                                                           uint32_t* __restrict__ ranks,
                                                           int64_t* __restrict__ ids) {
    __shared__ uint32_t tot[kBlock / kWave];
    const int64_t n = *valid, base = static_cast<int64_t>(blockIdx.x) * (kBlock * kPer);
    uint32_t part = 0, before;
    for (uint32_t k = threadIdx.x; k < blockIdx.x; k += kBlock) part += heads[k];
    block_prefix<kBlock>(part, tot, &before);
    const int64_t first = base + static_cast<int64_t>(threadIdx.x) * kPer;
    uint32_t is_head = 0;
    for (int s = 0; s < kPer; ++s) {
        const int64_t i = first + s;
        if (i < n && (i == 0 || keys[i - 1] != keys[i])) is_head |= 1u << s;
    }
    uint32_t all;
    uint32_t u = before + block_prefix<kBlock>(__popc(is_head), tot, &all);
    static_assert(kSpan % kPer == 0, "a span starts with a thread's places");
    if (first % kSpan == 0 && first < n) ranks[first / kSpan] = u;
    for (int s = 0; s < kPer; ++s)
        if ((is_head >> s) & 1) ids[u++] = keys[first + s];
}

// ------------------------------------------------------------- host side

size_t round256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

struct SortLayout {
    int passes, bits;  // of a pass's digit
    int items;         // keys a thread
    uint32_t tiles;
    bool small;
    size_t keys[2], places[2], counts, totals, bad, valid, heads, ranks, bytes;
};

SortLayout sort_layout(int64_t num_rows, int64_t count, bool sparse) {
    SortLayout l{};
    const int all = bits_below(num_rows);
    l.passes = all <= kDigitBits ? 1 : (all + kDigitBits - 1) / kDigitBits;
    l.bits = all == 0 ? 1 : (all + l.passes - 1) / l.passes;
    l.items = count <= int64_t{kFlatTiles} * kBlock * kFewItems ? kFewItems : kItems;
    const int64_t tile = kBlock * l.items;
    l.tiles = static_cast<uint32_t>(count > 0 ? (count + tile - 1) / tile : 1);
    l.small = count <= kSmallPlaces;
    size_t at = 0;
    auto take = [&at](size_t bytes) {
        const size_t a = at;
        at += round256(bytes);
        return a;
    };
    for (int b = 0; b < (l.small ? 1 : 2); ++b) {
        l.keys[b] = take(static_cast<size_t>(count) * 4);
        l.places[b] = take(static_cast<size_t>(count) * 4);
    }
    l.valid = take(4);
    if (!l.small) {
        l.counts = take(static_cast<size_t>(l.tiles) * kDigits * 4);
        l.totals = take(kDigits * 4);
        l.bad = take(static_cast<size_t>(l.tiles) * 4);
    }
    if (sparse) {
        if (!l.small) l.heads = take(static_cast<size_t>(l.tiles) * 4);
        l.ranks = take(static_cast<size_t>((count + kSpan - 1) / kSpan) * 4);
    }
    l.bytes = at;
    return l;
}

// Blocks of `threads` threads that clear, none only of nothing (one clears what
// lies before and after the whole packs): 512 threads a compute unit, whose stores
// stay near each other (714 MB: 6.1 TB/s, with 2,048 threads 4.1).
unsigned clear_blocks(const ClearOut& c, int threads, int cus) {
    const size_t stores = (c.bytes + 15) / 16 + static_cast<size_t>(c.num_ids);
    const size_t per = static_cast<size_t>(threads) * 4, most = static_cast<size_t>(cus) * 512 / threads;
    const size_t b = (stores + per - 1) / per;
    return static_cast<unsigned>(b < most ? b : most);
}

// Part k of n of what there is to clear (the ids all in the first): the sort's
// launches are short and leave the memory idle, so each clears a part beside its
// work (2.65 M rows of 128 bfloat16 into 2^20: 353 us with all of it in the first, 318).
ClearOut clear_part(const ClearOut& c, int k, int n) {
    const size_t chunk = (c.bytes / n + 4096) & ~size_t{4095};
    const size_t from = chunk * k < c.bytes ? chunk * k : c.bytes;
    const size_t bytes = c.bytes - from < chunk ? c.bytes - from : chunk;
    return ClearOut{static_cast<unsigned char*>(c.p) + from, bytes, c.streamed, c.ids,
                    k == 0 ? c.num_ids : 0};
}

struct Words {  // of the workspace
    unsigned char* p;
    uint32_t* operator()(size_t at) const { return reinterpret_cast<uint32_t*>(p + at); }
};

template <int kPer>
int launch_passes(const Nodes& nodes, int64_t count, const ClearOut& clear, int64_t* work,
                  const Words& words, const SortLayout& l, int cus, SortedPlaces& sorted,
                  hipStream_t stream) {
    uint32_t* counts = words(l.counts);
    uint32_t* valid = words(l.valid);
    int cur = 0;
    for (int pass = 0; pass < l.passes; ++pass) {
        const bool first = pass == 0;
        const SortIn in{nodes, count, words(l.keys[cur]), words(l.places[cur]), valid,
                        pass * l.bits, l.bits};
        const int to = first ? 0 : cur ^ 1;
        const ClearOut in_count = clear_part(clear, 2 * pass, 2 * l.passes);
        const ClearOut in_scatter = clear_part(clear, 2 * pass + 1, 2 * l.passes);
        auto* count_kernel = first ? digit_count_kernel<true, kPer> : digit_count_kernel<false, kPer>;
        hipLaunchKernelGGL(count_kernel, dim3(l.tiles + clear_blocks(in_count, kBlock, cus)),
                           dim3(kBlock), 0, stream, in, l.tiles, counts, words(l.bad), in_count);
        MLXC_HIP_TRY(hipGetLastError());
        if (l.tiles > kFlatTiles) {
            hipLaunchKernelGGL(digit_prefix_kernel, dim3(kDigits), dim3(kBlock), 0, stream, counts,
                               l.tiles, words(l.totals));
            MLXC_HIP_TRY(hipGetLastError());
        }
        auto* scatter =
            first ? digit_scatter_kernel<true, kPer> : digit_scatter_kernel<false, kPer>;
        hipLaunchKernelGGL(scatter, dim3(l.tiles + clear_blocks(in_scatter, kBlock, cus)),
                           dim3(kBlock), 0, stream, in, l.tiles, counts, words(l.totals),
                           words(l.bad), words(l.keys[to]), words(l.places[to]), valid, work,
                           in_scatter);
        MLXC_HIP_TRY(hipGetLastError());
        cur = to;
    }
    sorted.keys = words(l.keys[cur]);
    sorted.places = words(l.places[cur]);
    if (!sorted.ranks) return MLXC_OK;
    hipLaunchKernelGGL(count_heads_kernel<kPer>, dim3(l.tiles), dim3(kBlock), 0, stream, sorted.keys,
                       valid, words(l.heads));
    MLXC_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(list_runs_kernel<kPer>, dim3(l.tiles), dim3(kBlock), 0, stream, sorted.keys,
                       valid, words(l.heads), words(l.ranks), clear.ids);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

}  // namespace

size_t place_sort_bytes(int64_t num_rows, int64_t count, bool sparse) {
    return sort_layout(num_rows, count, sparse).bytes;
}

int launch_place_sort(const Nodes& nodes, int64_t count, const ClearOut& clear, int64_t* work,
                      void* workspace, SortedPlaces& sorted, hipStream_t stream) {
    const bool sparse = clear.ids != nullptr;
    const SortLayout l = sort_layout(nodes.num_rows, count, sparse);
    DeviceInfo info;
    if (int rc = device_info(info)) return rc;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    const Words words{ws};
    uint32_t* valid = words(l.valid);
    uint32_t* ranks = sparse ? words(l.ranks) : nullptr;
    if (l.small) {
        hipLaunchKernelGGL(sort_small_kernel, dim3(1 + clear_blocks(clear, kSmallThreads, info.cus)),
                           dim3(kSmallThreads), 0, stream, nodes, static_cast<int32_t>(count), l.bits,
                           l.passes, clear, words(l.keys[0]), words(l.places[0]), valid, ranks, work);
        MLXC_HIP_TRY(hipGetLastError());
        sorted = SortedPlaces{words(l.keys[0]), words(l.places[0]), valid, ranks};
        return MLXC_OK;
    }
    sorted = SortedPlaces{nullptr, nullptr, valid, ranks};
    return l.items == kItems
               ? launch_passes<kItems>(nodes, count, clear, work, words, l, info.cus, sorted, stream)
               : launch_passes<kFewItems>(nodes, count, clear, work, words, l, info.cus, sorted,
                                          stream);
}

}  // namespace mlxc
