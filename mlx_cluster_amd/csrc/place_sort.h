// Device helpers of the sorts by node (place_sort.hip, embedding.hip).
#pragma once

#include "train_host.h"

namespace mlxc {

namespace {

constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kItems = 16;              // keys a thread

// Lists that one block takes, in LDS.
constexpr int kSmallThreads = 1024;
constexpr int kSmallPlaces = kSmallThreads * kItems;
constexpr int kSmallWaves = kSmallThreads / kWave;

// Exclusive prefix of one value a thread over the block; *total the sum.  `tot`
// is kThreads / 64 words of LDS.  Contains two barriers.
template <int kThreads>
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
#pragma unroll
    for (int k = 0; k < kThreads / kWave; ++k) {
        if (k < w) before += tot[k];
        all += tot[k];
    }
    *total = all;
    __syncthreads();
    return before + inc - v;
}

// Lanes of the wavefront that are active and hold this lane's digit of `bits`
// bits.  A bit's ballot m and the lane's own bit e, as 0 or ~0, differ in the
// lanes that m ^ e marks; what no bit marks is left.  differ | (m ^ e) is one
// instruction a half (table 0xbe over (m, e, differ)), so a bit costs four.
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool active) {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
        if (b >= bits) break;
        const uint32_t e = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int32_t>(d), b, 1));
        const uint64_t m = __builtin_amdgcn_uicmp(e, 0u, 33);  // 33: not equal
        lo = __builtin_amdgcn_bitop3_b32(static_cast<uint32_t>(m), e, lo, 0xbe);
        hi = __builtin_amdgcn_bitop3_b32(static_cast<uint32_t>(m >> 32), e, hi, 0xbe);
    }
    return __ballot(active) & ~(static_cast<uint64_t>(hi) << 32 | lo);
}

// One slot's rank among the keys of its digit before it in the wavefront's
// stretch, whose counts so far are cnt[digit].
__device__ __forceinline__ uint32_t take_rank(uint32_t* cnt, uint32_t d, int bits, bool active) {
    const uint64_t peers = same_digit(d, bits, active);
    const uint32_t before = cnt[d];
    const int r = lane_rank(peers);
    // the first of the peers writes after all of them have read (one
    // wavefront: in order)
    if (active && r == 0) cnt[d] = before + __popcll(peers);
    __builtin_amdgcn_wave_barrier();
    return before + r;
}

// Nodes base + s * stride (s < kCount) of a list of n, -1 past its end and where
// there is none.  Every load is issued before a value is used: past the end the
// last node again, so that no load sits behind a branch, which the compiler waits
// at (the first move of four lists of 48,100 to 5.3 M places: 21.4 -> 17.9 us on
// average).
template <int kCount>
__device__ __forceinline__ void load_nodes(int32_t (&v)[kCount], const Nodes& nodes, int64_t base,
                                           int stride, int64_t n, bool& bad) {
    int64_t raw[kCount];
    if (nodes.wide) {
        const int64_t* p = static_cast<const int64_t*>(nodes.p);
#pragma unroll
        for (int s = 0; s < kCount; ++s) {
            const int64_t i = base + static_cast<int64_t>(s) * stride;
            raw[s] = n > 0 ? p[i < n ? i : n - 1] : -1;
        }
    } else {
        const int32_t* p = static_cast<const int32_t*>(nodes.p);
#pragma unroll
        for (int s = 0; s < kCount; ++s) {
            const int64_t i = base + static_cast<int64_t>(s) * stride;
            raw[s] = n > 0 ? p[i < n ? i : n - 1] : -1;
        }
    }
#pragma unroll
    for (int s = 0; s < kCount; ++s) {
        const bool ok = static_cast<uint64_t>(raw[s]) < static_cast<uint64_t>(nodes.num_rows);
        bad |= !ok && raw[s] != -1;
        v[s] = ok && base + static_cast<int64_t>(s) * stride < n ? static_cast<int32_t>(raw[s]) : -1;
    }
}

// Pass `pass` of a sort of n entries in LDS by one block: a stable sort of keys
// and places by the digit of `bits` bits at pass * bits.  Entry base + s *
// kWave of a thread (s < items) is key[s], place[s] where `have` says so; n is
// then the number of entries that are.  Called by all threads; ends with a
// barrier.
struct SmallSort {
    uint32_t keys[kSmallPlaces];
    uint16_t places[kSmallPlaces];
    uint32_t cnt[kSmallWaves][kDigits];
    uint32_t tot[kSmallWaves];
};
static_assert(kSmallPlaces <= 65536, "places in 16 bits");

__device__ __forceinline__ void small_pass(SmallSort& l, const uint32_t (&key)[kItems],
                                           const uint32_t (&place)[kItems], uint32_t have,
                                           int items, int from, int bits, int32_t& n) {
    const int t = threadIdx.x, w = t / kWave;
    const uint32_t mask = (1u << bits) - 1;
    uint32_t rank[kItems];
    for (int k = t; k < kSmallWaves * kDigits; k += kSmallThreads) (&l.cnt[0][0])[k] = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        if (s >= items) break;
        rank[s] = take_rank(l.cnt[w], (key[s] >> from) & mask, bits, (have >> s) & 1);
    }
    __syncthreads();
    uint32_t sum = 0;
    if (t < kDigits)
        for (int k = 0; k < kSmallWaves; ++k) sum += l.cnt[k][t];
    uint32_t all;
    uint32_t to = block_prefix<kSmallThreads>(sum, l.tot, &all);
    if (t < kDigits) {
        for (int k = 0; k < kSmallWaves; ++k) {
            const uint32_t c = l.cnt[k][t];
            l.cnt[k][t] = to;
            to += c;
        }
    }
    n = static_cast<int32_t>(all);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        if (!((have >> s) & 1)) continue;
        const uint32_t j = l.cnt[w][(key[s] >> from) & mask] + rank[s];
        l.keys[j] = key[s];
        l.places[j] = static_cast<uint16_t>(place[s]);
    }
    __syncthreads();
}

// A thread's entries of the n in LDS, for the next pass; returns which are.
__device__ __forceinline__ uint32_t small_entries(const SmallSort& l, uint32_t (&key)[kItems],
                                                  uint32_t (&place)[kItems], int32_t n, int& items) {
    items = (n + kSmallThreads - 1) / kSmallThreads;
    const int32_t base = threadIdx.x / kWave * items * kWave + threadIdx.x % kWave;
    uint32_t have = 0;
#pragma unroll
    for (int s = 0; s < kItems; ++s) {
        if (s >= items) break;
        const int32_t i = base + s * kWave;
        have |= static_cast<uint32_t>(i < n) << s;
        key[s] = l.keys[i < n ? i : 0];
        place[s] = l.places[i < n ? i : 0];
    }
    return have;
}

// Bits of n - 1.
inline int bits_below(int64_t n) {
    int b = 0;
    for (uint64_t x = n > 1 ? static_cast<uint64_t>(n - 1) : 0; x; x >>= 1) ++b;
    return b;
}

}  // namespace

}  // namespace mlxc
