// Preference loss of paired log ratios, and its gradients.
//
// For a pair with r = the sum (or mean) of values - reference over the places
// that a side's mask leaves, z = beta * (r_chosen - r_rejected):
//   loss      (1 - e) softplus(-z) + e softplus(z),  softplus(x) = max(x, 0) + log1p(exp(-|x|))
//   d loss/dz -(1 - e) sigma(-z) + e sigma(z)
// and a value's gradient is d loss/dz * beta (/ its side's count), negated on
// the rejected side, 0 where it is masked.  A term whose weight is 0 is left
// out, so that an infinite z does not meet it.
#include "train_host.h"

namespace mlxc {

namespace {

constexpr int kWaves = kBlock / kWave;

struct Side {
    const void* values;
    const void* reference;
    const uint8_t* mask;
    int64_t length;
    void* grad;
};

struct PairTerms {
    float loss, slope;  // slope: d loss / d z
};

// softplus and sigma of z and -z from one exponential, one logarithm and one
// division: with e = exp(-|z|), softplus(+-z) = max(+-z, 0) + log1p(e), and the
// sigmas are 1 / (1 + e) and e / (1 + e).
__device__ __forceinline__ PairTerms pair_terms(float z, float smoothing) {
    const float e = expf(-fabsf(z));
    const float log_term = log1pf(e), large = 1.f / (1.f + e), small = e * large;
    const float up = z >= 0.f ? large : small, down = z >= 0.f ? small : large;  // sigma(z), sigma(-z)
    PairTerms t{0.f, 0.f};
    if (smoothing < 1.f) {
        t.loss += (1.f - smoothing) * (fmaxf(-z, 0.f) + log_term);
        t.slope -= (1.f - smoothing) * down;
    }
    if (smoothing > 0.f) {
        t.loss += smoothing * (fmaxf(z, 0.f) + log_term);
        t.slope += smoothing * up;
    }
    return t;
}

// x, or 0 where bit i of `bits` is clear.
__device__ __forceinline__ float keep_bit(float x, uint32_t bits, int i) {
    return __builtin_bit_cast(float, __builtin_bit_cast(int32_t, x) &
                                         __builtin_amdgcn_sbfe(static_cast<int32_t>(bits), i, 1));
}

// The bytes of a pack that are not 0, one bit each.
template <int N>
__device__ __forceinline__ uint32_t set_bytes(const Pack<uint8_t, N>& m) {
    uint32_t bits = 0;
    if constexpr (N % 4 == 0) {
        typedef uint32_t Words __attribute__((ext_vector_type(N / 4)));
        uint32_t w[N / 4];
        if constexpr (N == 4) {
            w[0] = __builtin_bit_cast(uint32_t, m);
        } else {
            const Words words = __builtin_bit_cast(Words, m);
#pragma unroll
            for (int k = 0; k < N / 4; ++k) w[k] = words[k];
        }
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            // bit 7 of every byte that is not 0, gathered into 4 bits
            const uint32_t high = (((w[k] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[k]) >> 7 & 0x01010101u;
            bits |= (high * 0x01020408u >> 24 & 15u) << (4 * k);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) bits |= static_cast<uint32_t>(m.v[i] != 0) << i;
    }
    return bits;
}

// A group of 2^log lanes takes a pair.  A side's row lies anywhere in the packs
// of kPer elements (16 bytes, or one element where the arrays are not aligned):
// its lanes read the packs that it touches, and leave out what is not its own.
// A pair's row in its packs: element r (from `skip` elements before the row on)
// is at index base + r; the row is r in [skip, skip + length), the array ends
// at r = room.
struct RowView {
    int64_t base;
    int32_t skip, end, room;  // (lengths are below 2^30)
};
template <int kPer>
__device__ __forceinline__ RowView row_view(const Side& s, int64_t p, int64_t pairs) {
    const int64_t begin = p * s.length;
    RowView v;
    v.skip = static_cast<int32_t>(begin % kPer);
    v.base = begin - v.skip;
    v.end = v.skip + static_cast<int32_t>(s.length);
    const int64_t room = (pairs - p) * s.length + v.skip;
    v.room = static_cast<int32_t>(room < INT32_MAX ? room : INT32_MAX);
    return v;
}

// The places of the pack at element r that belong to the row and are not
// masked, one bit each.
template <int kPer>
__device__ __forceinline__ uint32_t own_places(const uint8_t* __restrict__ mask, const RowView& v,
                                               int32_t r) {
    const int32_t from = v.skip > r ? v.skip - r : 0;
    const int32_t to = v.end - r < kPer ? (v.end > r ? v.end - r : 0) : kPer;
    uint32_t own = from < to ? (1u << to) - (1u << from) : 0u;
    if (mask) {
        Pack<uint8_t, kPer> m;
        if (r + kPer <= v.room) {
            m = *reinterpret_cast<const Pack<uint8_t, kPer>*>(mask + v.base + r);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) m.v[i] = r + i < v.room ? mask[v.base + r + i] : 0;
        }
        own &= set_bytes(m);
    }
    return own;
}

// The pack at element r < v.room; past the array's end its last element.
template <typename E, int kPer>
__device__ __forceinline__ Pack<typename E::S, kPer> load_inside(
    const typename E::S* __restrict__ x, const RowView& v, int32_t r) {
    if (r + kPer <= v.room)
        return *reinterpret_cast<const Pack<typename E::S, kPer>*>(x + v.base + r);
    Pack<typename E::S, kPer> p;
#pragma unroll
    for (int i = 0; i < kPer; ++i) p.v[i] = x[v.base + (r + i < v.room ? r + i : v.room - 1)];
    return p;
}

struct RowSum {
    float sum, left;
};

// This lane's share of a pair's side: the sum of values - reference, and how
// many are left.  One pack at a time: more in flight cost registers, and with
// them wavefronts (two: 131 registers, 3 wavefronts a SIMD, and 39 us instead of 33 for
// the 4,097 ragged pairs below).
template <typename E, int kPer>
__device__ __forceinline__ RowSum row_share(const Side& s, int64_t p, int64_t pairs, int lane,
                                            int lanes) {
    using S = typename E::S;
    const RowView view = row_view<kPer>(s, p, pairs);
    const S* values = static_cast<const S*>(s.values);
    const S* reference = static_cast<const S*>(s.reference);
    RowSum sum{0.f, 0.f};
    for (int32_t r = lane * kPer; r < view.end; r += lanes * kPer) {
        const Pack<S, kPer> v = load_inside<E, kPer>(values, view, r);
        Pack<S, kPer> f;
        if (reference) f = load_inside<E, kPer>(reference, view, r);
        const uint32_t own = own_places<kPer>(s.mask, view, r);
        sum.left += static_cast<float>(__popc(own));
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float d = E::load(v.v[i]) - (reference ? E::load(f.v[i]) : 0.f);
            sum.sum += keep_bit(d, own, i);
        }
    }
    return sum;
}

// Writes a row of a side's gradient.
template <typename E, int kPer>
__device__ __forceinline__ void grad_row(const Side& s, int64_t p, int64_t pairs, float slope,
                                         int lane, int lanes) {
    using S = typename E::S;
    const RowView view = row_view<kPer>(s, p, pairs);
    S* grad = static_cast<S*>(s.grad) + view.base;
    const S value = E::store(slope);
    for (int32_t r = lane * kPer; r < view.end; r += lanes * kPer) {
        const uint32_t own = own_places<kPer>(s.mask, view, r);
        Pack<S, kPer> g;
#pragma unroll
        for (int i = 0; i < kPer; ++i) g.v[i] = (own >> i) & 1 ? value : S(0);
        if (r >= view.skip && r + kPer <= view.end) {
            *reinterpret_cast<Pack<S, kPer>*>(grad + r) = g;
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (r + i >= view.skip && r + i < view.end) grad[r + i] = g.v[i];
        }
    }
}

__device__ __forceinline__ float wave_sum(float x, int lanes = kWave) {
    for (int o = lanes / 2; o > 0; o >>= 1) x += __shfl_xor(x, o, kWave);
    return x;
}

// Sum over the block, valid in thread 0; `part` is kWaves words of LDS.
__device__ __forceinline__ float block_sum(float x, float* part) {
    x = wave_sum(x);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = x;
    __syncthreads();
    float all = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all += part[k];
    return all;
}

// partial[block] <- the sum of the block's pairs' losses.
template <typename E, int kPer>
__global__ __launch_bounds__(kBlock) void preference_kernel(Side chosen, Side rejected,
                                                            int64_t pairs, int log, float beta,
                                                            float smoothing, bool normalize,
                                                            float share, float* __restrict__ rewards,
                                                            float* __restrict__ slopes,
                                                            float* __restrict__ partial) {
    __shared__ float part[kWaves];
    const int lanes = 1 << log;
    const int lane = threadIdx.x & (lanes - 1);
    const int per_block = kBlock >> log;
    float loss = 0.f;
    for (int64_t p = blockIdx.x * static_cast<int64_t>(per_block) + (threadIdx.x >> log); p < pairs;
         p += static_cast<int64_t>(gridDim.x) * per_block) {
        const RowSum c = row_share<E, kPer>(chosen, p, pairs, lane, lanes);
        const RowSum d = row_share<E, kPer>(rejected, p, pairs, lane, lanes);
        float per_c = 1.f, per_d = 1.f;
        if (normalize) {
            per_c = 1.f / fmaxf(wave_sum(c.left, lanes), 1.f);
            per_d = 1.f / fmaxf(wave_sum(d.left, lanes), 1.f);
        }
        const float rc = beta * (wave_sum(c.sum, lanes) * per_c);
        const float rd = beta * (wave_sum(d.sum, lanes) * per_d);
        const PairTerms t = pair_terms(rc - rd, smoothing);
        const float dz = t.slope * beta * share;
        if (lane == 0) {
            loss += t.loss;
            if (rewards) {
                rewards[p] = rc;
                rewards[pairs + p] = rd;
            }
            if (slopes) {
                slopes[p] = dz * per_c;
                slopes[pairs + p] = -dz * per_d;
            }
        }
        if (chosen.grad) grad_row<E, kPer>(chosen, p, pairs, dz * per_c, lane, lanes);
        if (rejected.grad) grad_row<E, kPer>(rejected, p, pairs, -dz * per_d, lane, lanes);
    }
    loss = block_sum(loss, part);
    if (threadIdx.x == 0) partial[blockIdx.x] = loss;
}

// Long rows: a block a pair, half of it a side.  4,097 pairs of 777 and 1,025 ragged
// bfloat16 under masks (52 MB) take 26 us, 13 of them vector instructions.
template <typename E, int kPer>
__global__ __launch_bounds__(kBlock) void preference_long_kernel(
    Side chosen, Side rejected, int64_t pairs, int, float beta, float smoothing, bool normalize,
    float share, float* __restrict__ rewards, float* __restrict__ slopes,
    float* __restrict__ partial) {
    constexpr int kHalf = kBlock / 2;
    __shared__ float sums[kWaves], lefts[kWaves];
    const int t = threadIdx.x, lane = t % kHalf, w = t / kWave;
    const int half = __builtin_amdgcn_readfirstlane(t / kHalf);  // the same in a wavefront
    const Side& s = half ? rejected : chosen;
    float loss = 0.f;
    for (int64_t p = blockIdx.x; p < pairs; p += gridDim.x) {
        const RowSum x = row_share<E, kPer>(s, p, pairs, lane, kHalf);
        const float sum = wave_sum(x.sum), left = wave_sum(x.left);
        if (t % kWave == 0) {
            sums[w] = sum;
            lefts[w] = left;
        }
        __syncthreads();
        float r[2], per[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float all = 0.f, kept = 0.f;
#pragma unroll
            for (int k = 0; k < kWaves / 2; ++k) {
                all += sums[h * (kWaves / 2) + k];
                kept += lefts[h * (kWaves / 2) + k];
            }
            per[h] = normalize ? 1.f / fmaxf(kept, 1.f) : 1.f;
            r[h] = beta * (all * per[h]);
        }
        const PairTerms terms = pair_terms(r[0] - r[1], smoothing);
        const float dz = terms.slope * beta * share;
        const float slope = half ? -dz * per[1] : dz * per[0];
        if (t == 0) loss += terms.loss;
        if (lane == 0) {
            if (rewards) rewards[half * pairs + p] = r[half];
            if (slopes) slopes[half * pairs + p] = slope;
        }
        if (s.grad) grad_row<E, kPer>(s, p, pairs, slope, lane, kHalf);
        __syncthreads();
    }
    if (t == 0) partial[blockIdx.x] = loss;
}

// Short rows: a block takes kBlock >> log pairs at a time, 2^log threads a pair.
// Their rows are one stretch of each array, read and written in whole packs by
// all threads; the differences pass through LDS to the threads that add them
// up (rows there an odd number of words apart), the slopes back.
//
// Bound by the stream of the values, references and gradients: of 9 float32 a
// side, 4.7 M pairs (1.06 GB) 207 us, as long as a copy of those bytes.  A group of
// lanes a pair, over the packs that its rows touch, takes 531 us: the packs' edges
// and every lane's own exponentials keep the vector units busy.
constexpr int kShortLength = 64;
constexpr int kShortWords = kBlock * (kShortLength / 4 + 1);

struct Divide {  // e / length for e < 2^16
    uint32_t length, inverse;
    __device__ __forceinline__ explicit Divide(uint32_t n)
        : length(n), inverse(n > 1 ? 0xffffffffu / n + 1 : 0) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t e) const {
        return length > 1 ? __umulhi(e, inverse) : e;
    }
};

// Calls f(element, row, column, bit) for the elements of a pack at e that lie
// below n; `mask`: with their mask's bytes, from the stretch's first.
template <int kPer, typename F>
__device__ __forceinline__ void each_of_pack(const uint8_t* __restrict__ mask, uint32_t e,
                                             uint32_t n, const Divide& rows, F f) {
    Pack<uint8_t, kPer> m;
    if (mask) {
        if (e + kPer <= n) {
            m = *reinterpret_cast<const Pack<uint8_t, kPer>*>(mask + e);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) m.v[i] = e + i < n ? mask[e + i] : 0;
        }
    }
    uint32_t row = rows(e), col = e - row * rows.length;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        f(i, row, col, !mask || m.v[i]);
        if (++col == rows.length) {
            col = 0;
            ++row;
        }
    }
}

template <typename E, int kPer>
__global__ __launch_bounds__(kBlock) void preference_short_kernel(
    Side chosen, Side rejected, int64_t pairs, int log, float beta, float smoothing, bool normalize,
    float share, float* __restrict__ rewards, float* __restrict__ slopes,
    float* __restrict__ partial) {
    using S = typename E::S;
    __shared__ float diff[kShortWords];
    __shared__ uint8_t kept[kShortWords];
    __shared__ float slope[2][kBlock];
    __shared__ float part[kWaves];
    const int t = threadIdx.x, per_block = kBlock >> log, parts = 1 << log;
    const int own = t >> log, share_of = t & (parts - 1);  // the thread's pair, and part of it
    float loss = 0.f;
    for (int64_t p0 = blockIdx.x * static_cast<int64_t>(per_block); p0 < pairs;
         p0 += static_cast<int64_t>(gridDim.x) * per_block) {
        const int count = pairs - p0 < per_block ? static_cast<int>(pairs - p0) : per_block;
        float r[2], per[2];
        for (int side = 0; side < 2; ++side) {
            const Side& s = side ? rejected : chosen;
            const uint32_t length = static_cast<uint32_t>(s.length), n = count * length;
            const uint32_t pitch = length | 1;
            const Divide rows(length);
            const S* values = static_cast<const S*>(s.values) + p0 * s.length;
            const S* reference =
                s.reference ? static_cast<const S*>(s.reference) + p0 * s.length : nullptr;
            const uint8_t* mask = s.mask ? s.mask + p0 * s.length : nullptr;
            for (uint32_t e = t * kPer; e < n; e += kBlock * kPer) {
                float d[kPer];
                if (e + kPer <= n) {
                    load_pack<E, kPer>(d, values + e);
                    if (reference) {
                        float f[kPer];
                        load_pack<E, kPer>(f, reference + e);
#pragma unroll
                        for (int i = 0; i < kPer; ++i) d[i] -= f[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const uint32_t at = e + i < n ? e + i : n - 1;
                        d[i] = E::load(values[at]) - (reference ? E::load(reference[at]) : 0.f);
                    }
                }
                each_of_pack<kPer>(mask, e, n, rows, [&](int i, uint32_t row, uint32_t col, bool in) {
                    if (e + i >= n) return;
                    diff[row * pitch + col] = in ? d[i] : 0.f;
                    if (mask) kept[row * pitch + col] = in;
                });
            }
            __syncthreads();
            float sum = 0.f, left = mask ? 0.f : static_cast<float>(length);
            if (own < count) {
                for (uint32_t c = share_of; c < length; c += parts) sum += diff[own * pitch + c];
                if (mask && normalize)
                    for (uint32_t c = share_of; c < length; c += parts)
                        left += kept[own * pitch + c];
            }
            for (int o = parts / 2; o > 0; o >>= 1) {
                sum += __shfl_xor(sum, o, kWave);
                if (mask) left += __shfl_xor(left, o, kWave);
            }
            per[side] = normalize ? 1.f / fmaxf(left, 1.f) : 1.f;
            r[side] = beta * (sum * per[side]);
            __syncthreads();
        }
        if (own < count && share_of == 0) {
            const PairTerms terms = pair_terms(r[0] - r[1], smoothing);
            loss += terms.loss;
            const float dz = terms.slope * beta * share;
            slope[0][own] = dz * per[0];
            slope[1][own] = -dz * per[1];
            if (rewards) {
                rewards[p0 + own] = r[0];
                rewards[pairs + p0 + own] = r[1];
            }
            if (slopes) {
                slopes[p0 + own] = dz * per[0];
                slopes[pairs + p0 + own] = -dz * per[1];
            }
        }
        __syncthreads();
        for (int side = 0; side < 2; ++side) {
            const Side& s = side ? rejected : chosen;
            if (!s.grad) continue;
            const uint32_t length = static_cast<uint32_t>(s.length), n = count * length;
            const Divide rows(length);
            S* grad = static_cast<S*>(s.grad) + p0 * s.length;
            const uint8_t* mask = s.mask ? s.mask + p0 * s.length : nullptr;
            for (uint32_t e = t * kPer; e < n; e += kBlock * kPer) {
                float g[kPer];
                each_of_pack<kPer>(mask, e, n, rows, [&](int i, uint32_t row, uint32_t, bool in) {
                    g[i] = e + i < n && in ? slope[side][row] : 0.f;
                });
                if (e + kPer <= n) {
                    store_pack<E, kPer>(grad + e, g);
                } else {
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (e + i < n) grad[e + i] = E::store(g[i]);
                }
            }
        }
        __syncthreads();
    }
    loss = block_sum(loss, part);
    if (t == 0) partial[blockIdx.x] = loss;
}

// *loss <- share * the sum of n partial sums, in a fixed order.
__global__ __launch_bounds__(kBlock) void loss_sum_kernel(const float* __restrict__ partial, int n,
                                                          float share, float* __restrict__ loss) {
    __shared__ float part[kWaves];
    float s = 0.f;
    for (int k = threadIdx.x; k < n; k += kBlock) s += partial[k];
    s = block_sum(s, part);
    if (threadIdx.x == 0) *loss = s * share;
}

// 2^log lanes a pair and side, or (log = 8) the block.
template <typename E, int kPer>
__global__ __launch_bounds__(kBlock) void preference_grad_kernel(Side chosen, Side rejected,
                                                                 int64_t pairs, int log,
                                                                 const float* __restrict__ slopes,
                                                                 const float* upstream) {
    const int lanes = 1 << log;
    const int lane = threadIdx.x & (lanes - 1);
    const int per_block = kBlock >> log;
    const float up = upstream ? *upstream : 1.f;
    const Side& s = blockIdx.y ? rejected : chosen;
    if (!s.grad) return;
    for (int64_t p = blockIdx.x * static_cast<int64_t>(per_block) + (threadIdx.x >> log); p < pairs;
         p += static_cast<int64_t>(gridDim.x) * per_block)
        grad_row<E, kPer>(s, p, pairs, up * slopes[blockIdx.y * pairs + p], lane, lanes);
}

// ------------------------------------------------------------- host side

Side side(const mlxc_preference_side& s) {
    return Side{s.values, s.reference, s.mask, s.length, s.grad};
}

constexpr int kMaxBlocks = 4096;
// Short rows: the blocks that are resident together (their LDS), so that their
// stretches stay near each other (4.7 M pairs of 9: 204 us, 208 with 4,096 blocks).
constexpr int kShortBlocksPerUnit = 6;

enum class Rows { kShort, kGroup, kLong };

// How a call is spread: its kernel, 2^log threads a pair, and the blocks.
struct Spread {
    Rows rows;
    int log;
    int blocks;
    bool packed;  // whole packs: every array 16-byte aligned (a mask its share of it)
};

// The kernel goes by the longer side.  Up to kShortLength values the rows pass
// through LDS; a row that more than a wavefront's packs reach takes half a
// block; a group of lanes takes those between.
int spread(const PreferenceCall& c, Spread& s) {
    s = Spread{};
    const size_t esz = elem_bytes(c.dtype);
    const int64_t per = 16 / esz;
    int64_t longest = 1;
    s.packed = true;
    for (const mlxc_preference_side& x : c.side) {
        const uintptr_t all = reinterpret_cast<uintptr_t>(x.values) |
                              reinterpret_cast<uintptr_t>(x.reference) |
                              reinterpret_cast<uintptr_t>(x.grad);
        if (all % 16 != 0 || reinterpret_cast<uintptr_t>(x.mask) % per != 0) s.packed = false;
        if (x.length > longest) longest = x.length;
    }
    const int64_t packs = s.packed ? (longest + 2 * per - 2) / per : longest;  // of a row at most
    if (longest <= kShortLength) {
        s.rows = Rows::kShort;
        while ((16 << s.log) < longest) ++s.log;  // 16 values a thread
    } else if (packs > kWave) {
        s.rows = Rows::kLong;
        s.log = 8;
    } else {
        s.rows = Rows::kGroup;
        while ((1 << s.log) < packs) ++s.log;
    }
    const int64_t b = (c.pairs + (kBlock >> s.log) - 1) / (kBlock >> s.log);
    int most = kMaxBlocks;
    if (s.rows == Rows::kShort) {
        DeviceInfo info;
        if (int rc = device_info(info)) return rc;
        if (info.cus * kShortBlocksPerUnit < most) most = info.cus * kShortBlocksPerUnit;
    }
    s.blocks = static_cast<int>(b < 1 ? 1 : b > most ? most : b);
    return MLXC_OK;
}

template <typename E, int kPer>
int loss_launch(const PreferenceCall& c, const Spread& s, float* loss, float* rewards,
                float* slopes, void* workspace, hipStream_t stream) {
    const float share = c.sum || c.pairs == 0 ? 1.f : static_cast<float>(1.0 / c.pairs);
    float* partial = static_cast<float*>(workspace);
    auto* kernel = s.rows == Rows::kShort   ? preference_short_kernel<E, kPer>
                   : s.rows == Rows::kGroup ? preference_kernel<E, kPer>
                                            : preference_long_kernel<E, kPer>;
    hipLaunchKernelGGL(kernel, dim3(s.blocks), dim3(kBlock), 0, stream, side(c.side[0]),
                       side(c.side[1]), c.pairs, s.log, c.beta, c.smoothing, c.normalize, share,
                       rewards, slopes, partial);
    MLXC_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(kBlock), 0, stream, partial, s.blocks, share,
                       loss);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E>
int loss_typed(const PreferenceCall& c, float* loss, float* rewards, float* slopes, void* workspace,
               hipStream_t stream) {
    constexpr int per = 16 / sizeof(typename E::S);
    Spread s;
    if (int rc = spread(c, s)) return rc;
    return s.packed ? loss_launch<E, per>(c, s, loss, rewards, slopes, workspace, stream)
                    : loss_launch<E, 1>(c, s, loss, rewards, slopes, workspace, stream);
}

template <typename E>
int grad_typed(const PreferenceCall& c, const float* slopes, const float* upstream,
               hipStream_t stream) {
    constexpr int per = 16 / sizeof(typename E::S);
    Spread s;
    if (int rc = spread(c, s)) return rc;
    // short rows: their packs a group
    const int log = s.rows == Rows::kShort ? s.log + 2 : s.log;
    const int64_t b = (c.pairs + (kBlock >> log) - 1) / (kBlock >> log);
    auto* kernel = s.packed ? preference_grad_kernel<E, per> : preference_grad_kernel<E, 1>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(b < kMaxBlocks ? b : kMaxBlocks), 2),
                       dim3(kBlock), 0, stream, side(c.side[0]), side(c.side[1]), c.pairs, log,
                       slopes, upstream);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

}  // namespace

size_t preference_workspace_bytes(int64_t pairs) {
    return static_cast<size_t>(pairs < 1 ? 1 : pairs > kMaxBlocks ? kMaxBlocks : pairs) *
           sizeof(float);
}

int launch_preference_loss(const PreferenceCall& c, float* loss, float* rewards, float* slopes,
                           void* workspace, hipStream_t stream) {
    if (c.dtype == MLXC_FLOAT32) return loss_typed<F32>(c, loss, rewards, slopes, workspace, stream);
    if (c.dtype == MLXC_BFLOAT16)
        return loss_typed<BF16>(c, loss, rewards, slopes, workspace, stream);
    return loss_typed<F16>(c, loss, rewards, slopes, workspace, stream);
}

int launch_preference_grad(const PreferenceCall& c, const float* slopes, const float* upstream,
                           hipStream_t stream) {
    if (c.pairs == 0) return MLXC_OK;
    if (c.dtype == MLXC_FLOAT32) return grad_typed<F32>(c, slopes, upstream, stream);
    if (c.dtype == MLXC_BFLOAT16) return grad_typed<BF16>(c, slopes, upstream, stream);
    return grad_typed<F16>(c, slopes, upstream, stream);
}

}  // namespace mlxc
