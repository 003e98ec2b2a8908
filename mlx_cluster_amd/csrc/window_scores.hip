// Scores of the skip-gram windows of walks, and their gradient by place.
//
// With U the rows of a walk's M nodes (zeros where there is no node), W = M -
// C + 1 windows and the band of the pairs (j, j + k), j < W, 1 <= k < C:
//   scores    S = s * the band of U U^T
//   gradient  dU = (D + D^T) U, D the band filled with the scores' gradients
// (the table's gradient adds dU up by node, embedding.hip).
//
// Both run on the matrix units, sixteen rows of a walk at a time, with the
// operands loaded from the table straight into the registers that the
// instructions read: no LDS, no barrier, every wavefront on its own.  Scores are
// bound by the gather of the rows: 65,536 walks of 81 nodes, 128 bfloat16, context
// 10 (1.36 GB of rows, 170 MB of scores) take 217 us, 6,100 with a wavefront a
// window and a dot product a pair on the vector units.
#include <type_traits>

#include "train_host.h"

namespace mlxc {

namespace {

constexpr int kWaves = kBlock / kWave;
constexpr int kTileRows = 16;  // rows (and columns) of a matrix instruction's result

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// How an element type meets the matrix unit.  A wavefront's lane holds kPer
// consecutive values of row lane % 16 in each step of kStep values: those from
// (lane / 16) * kPer on.  Both operands have that layout, so the registers of
// a tile of rows are either operand of a product of rows.
template <typename E>
struct Matrix;
template <>
struct Matrix<BF16> {
    static constexpr int kPer = 8, kStep = 32, kChains = 1;
    static __device__ __forceinline__ void mul(const Pack<uint16_t, 8>& a, const Pack<uint16_t, 8>& b,
                                               f32x4 (&c)[kChains]) {
        c[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c[0], 0, 0, 0);
    }
};
template <>
struct Matrix<F16> {
    static constexpr int kPer = 8, kStep = 32, kChains = 1;
    static __device__ __forceinline__ void mul(const Pack<_Float16, 8>& a, const Pack<_Float16, 8>& b,
                                               f32x4 (&c)[kChains]) {
        c[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c[0], 0, 0, 0);
    }
};
template <>
struct Matrix<F32> {
    static constexpr int kPer = 4, kStep = 16, kChains = 4;
    // one value of each lane an instruction: its four take the step's values
    // in another order, the same in both operands.  Each adds to a chain of its
    // own: one chain of dim sums was off by 2.0e-7 of the scores at dim 128, four by
    // 1.1e-7.
    static __device__ __forceinline__ void mul(const Pack<float, 4>& a, const Pack<float, 4>& b,
                                               f32x4 (&c)[kChains]) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            c[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[q], b.v[q], c[q], 0, 0, 0);
    }
};

// The sums of a product's chains.
template <typename E>
struct Chains {
    f32x4 c[Matrix<E>::kChains];
    __device__ __forceinline__ Chains() {
#pragma unroll
        for (int q = 0; q < Matrix<E>::kChains; ++q) c[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ f32x4 sum() const {
        if constexpr (Matrix<E>::kChains == 1) return c[0];
        else return (c[0] + c[1]) + (c[2] + c[3]);
    }
};

// kPer values of a row from value `at` on, zeros from dim on; `width` values
// (a power of two) lie aligned, dim is a multiple of it.
template <typename E, int kPer>
__device__ __forceinline__ Pack<typename E::S, kPer> load_values(const typename E::S* row,
                                                                 int32_t at, int32_t dim,
                                                                 int width) {
    using S = typename E::S;
    Pack<S, kPer> p;
#pragma unroll
    for (int q = 0; q < kPer; ++q) p.v[q] = S(0);
    auto pieces = [&](auto n) {
        constexpr int N = decltype(n)::value;
#pragma unroll
        for (int q = 0; q < kPer; q += N) {
            if (at + q < dim) {
                const Pack<S, N> x = *reinterpret_cast<const Pack<S, N>*>(row + at + q);
#pragma unroll
                for (int i = 0; i < N; ++i) p.v[q + i] = x.v[i];
            }
        }
    };
    if (width >= kPer) pieces(std::integral_constant<int, kPer>{});
    else if (width == 4) pieces(std::integral_constant<int, kPer < 4 ? kPer : 4>{});
    else if (width == 2) pieces(std::integral_constant<int, 2>{});
    else pieces(std::integral_constant<int, 1>{});
    return p;
}

// ------------------------------------------------------------- scores

template <typename E, int kSteps>
struct Fragment {
    Pack<typename E::S, Matrix<E>::kPer> v[kSteps];
};

// Values [from, from + kSteps * kStep) of this lane's row, zeros from dim on
// (which lies inside these steps wherever they are not all full, also between
// two of them).
// kAligned: packs of kPer values lie aligned and fill the rows, and the table
// has a row; without a branch then, and of no node the first row's.  Else
// zeros of no node.
template <typename E, int kSteps, bool kAligned>
__device__ __forceinline__ void load_fragment(Fragment<E, kSteps>& f,
                                              const typename E::S* __restrict__ weight,
                                              int64_t row_stride, int32_t dim, int width,
                                              int32_t node, int32_t from) {
    constexpr int kPer = Matrix<E>::kPer;
    const int lane = threadIdx.x % kWave;
    const typename E::S* row = weight + (node < 0 ? 0 : node) * row_stride;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int32_t at = from + s * Matrix<E>::kStep + lane / kTileRows * kPer;
        if (kAligned) {
            f.v[s] = *reinterpret_cast<const Pack<typename E::S, kPer>*>(row + (at < dim ? at : 0));
            if (from + kSteps * Matrix<E>::kStep > dim && at >= dim) {
#pragma unroll
                for (int q = 0; q < kPer; ++q) f.v[s].v[q] = 0;
            }
        } else {
            f.v[s] = load_values<E, kPer>(row, at, node < 0 ? 0 : dim, width);
        }
    }
}

// The node of row 16 * t + lane % 16 of a walk, -1 from M on.
__device__ __forceinline__ int32_t tile_node(const Walks& walks, int64_t n, int32_t t, bool& bad) {
    const int64_t i = static_cast<int64_t>(t) * kTileRows + threadIdx.x % kTileRows;
    return i < walks.walk_nodes
               ? static_cast<int32_t>(node_at(walks.nodes, n * walks.walk_nodes + i, bad))
               : -1;
}

// Scores of the pairs between row tile t (rows) and t + ahead (columns).
__device__ __forceinline__ void store_scores(const f32x4& acc, const Walks& walks, int64_t n,
                                             int32_t t, int ahead, uint32_t rows_valid,
                                             uint32_t cols_valid, float scale,
                                             float* __restrict__ scores) {
    const int lane = threadIdx.x % kWave;
    const int32_t W = static_cast<int32_t>(walks.windows());
    const int c = lane % kTileRows, r0 = lane / kTileRows * 4;
    // entry (j, k) is at (n * W + j) * (C - 1) + k - 1: from one row to the
    // next of the lane's column k falls by one
    float* first = scores + (n * W + t * kTileRows + r0) * (walks.ctx - 1) +
                   (ahead * kTileRows + c - r0 - 1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int r = r0 + q;
        const int k = ahead * kTileRows + c - r;
        if (t * kTileRows + r >= W || k < 1 || k >= walks.ctx) continue;
        const bool both = (rows_valid >> r) & (cols_valid >> c) & 1;
        first[static_cast<int64_t>(q) * (walks.ctx - 2)] = both ? acc[q] * scale : 0.f;
    }
}

// A wavefront's part of the call: row tiles [part * per, ...) of walk `walk`.
struct Split {
    int32_t parts;  // a walk's parts
    int32_t per;    // row tiles of a part
};

// A wavefront goes down a walk's row tiles: tile t's rows against its own and
// the kAhead tiles after it, which are all that C - 1 <= 16 * kAhead places
// reach, kept in registers until they are rows themselves; the next tile's
// loads fly meanwhile.  dim <= kSteps * kStep.
template <typename E, int kSteps, int kAhead, bool kAligned>
__global__ __launch_bounds__(kBlock) void window_scores_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, int32_t dim, int width,
    Walks walks, Split split, float scale, float* __restrict__ scores, int64_t* status) {
    const int32_t row_tiles = static_cast<int32_t>((walks.windows() + kTileRows - 1) / kTileRows);
    bool bad = false;
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave;
         u < walks.num_walks * split.parts; u += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t n = u / split.parts;
        const int32_t first = static_cast<int32_t>(u - n * split.parts) * split.per;
        const int32_t last = row_tiles - first > split.per ? first + split.per : row_tiles;
        Fragment<E, kSteps> f[kAhead + 1];
        uint32_t valid[kAhead + 1];
#pragma unroll
        for (int a = 0; a <= kAhead; ++a) {
            const int32_t node = tile_node(walks, n, first + a, bad);
            valid[a] = static_cast<uint32_t>(__ballot(node >= 0)) & 0xffffu;
            load_fragment<E, kSteps, kAligned>(f[a], weight, row_stride, dim, width, node, 0);
        }
        int32_t next_node = tile_node(walks, n, first + kAhead + 1, bad);
        for (int32_t t = first; t < last; ++t) {
            Fragment<E, kSteps> next;
            uint32_t next_valid = 0;
            if (t + 1 < last) {
                next_valid = static_cast<uint32_t>(__ballot(next_node >= 0)) & 0xffffu;
                load_fragment<E, kSteps, kAligned>(next, weight, row_stride, dim, width, next_node,
                                                   0);
                next_node = tile_node(walks, n, t + kAhead + 2, bad);
            }
#pragma unroll
            for (int a = 0; a <= kAhead; ++a) {
                Chains<E> acc;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) Matrix<E>::mul(f[0].v[s], f[a].v[s], acc.c);
                store_scores(acc.sum(), walks, n, t, a, valid[0], valid[a], scale, scores);
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                f[a] = f[a + 1];
                valid[a] = valid[a + 1];
            }
            f[kAhead] = next;
            valid[kAhead] = next_valid;
        }
    }
    report_bad(bad, status);
}

// Rows of any length: for every row tile, kSteps steps of all its tiles at a
// time.  A tile's rows are loaded again for the kAhead row tiles before it, as
// a rule from the caches.
template <typename E, int kSteps, int kAhead, bool kAligned>
__global__ __launch_bounds__(kBlock) void window_scores_long_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, int32_t dim, int width,
    Walks walks, Split split, float scale, float* __restrict__ scores, int64_t* status) {
    const int32_t row_tiles = static_cast<int32_t>((walks.windows() + kTileRows - 1) / kTileRows);
    bool bad = false;
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave;
         u < walks.num_walks * split.parts; u += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t n = u / split.parts;
        const int32_t first = static_cast<int32_t>(u - n * split.parts) * split.per;
        const int32_t last = row_tiles - first > split.per ? first + split.per : row_tiles;
        for (int32_t t = first; t < last; ++t) {
            int32_t node[kAhead + 1];
            Chains<E> acc[kAhead + 1];
#pragma unroll
            for (int a = 0; a <= kAhead; ++a) node[a] = tile_node(walks, n, t + a, bad);
            for (int32_t from = 0; from < dim; from += kSteps * Matrix<E>::kStep) {
                Fragment<E, kSteps> f[kAhead + 1];
#pragma unroll
                for (int a = 0; a <= kAhead; ++a)
                    load_fragment<E, kSteps, kAligned>(f[a], weight, row_stride, dim, width,
                                                       node[a], from);
#pragma unroll
                for (int a = 0; a <= kAhead; ++a)
#pragma unroll
                    for (int s = 0; s < kSteps; ++s)
                        Matrix<E>::mul(f[0].v[s], f[a].v[s], acc[a].c);
            }
            const uint32_t rows_valid = static_cast<uint32_t>(__ballot(node[0] >= 0)) & 0xffffu;
#pragma unroll
            for (int a = 0; a <= kAhead; ++a)
                store_scores(acc[a].sum(), walks, n, t, a, rows_valid,
                             static_cast<uint32_t>(__ballot(node[a] >= 0)) & 0xffffu, scale, scores);
        }
    }
    report_bad(bad, status);
}

// ------------------------------------------------------------- gradient by place

// Entry (i, o) of the walk's symmetric band: the gradient of the score between
// places i and o, 0 where they are no pair.
__device__ __forceinline__ float band_entry(const float* __restrict__ grad, const Walks& walks,
                                            int64_t n, int64_t i, int64_t o) {
    const int64_t j = i < o ? i : o, k = i < o ? o - i : i - o;
    const int64_t W = walks.windows();
    if (k < 1 || k >= walks.ctx || j < 0 || j >= W) return 0.f;
    return grad[(n * W + j) * (walks.ctx - 1) + k - 1];
}

// A tile's gradients without the matrix unit: only the band's own products.
template <typename E>
__device__ __forceinline__ void band_rows(const float* __restrict__ grad,
                                       const typename E::S* __restrict__ weight, int64_t row_stride,
                                       int32_t dim, const Walks& walks, int64_t n, int64_t i0,
                                       int32_t col0, int32_t cols, float* __restrict__ rows) {
    const int lane = threadIdx.x % kWave;
    const int64_t M = walks.walk_nodes;
    for (int64_t i = i0; i < i0 + kTileRows && i < M; ++i) {
        bool bad = false;
        const bool own = node_at(walks.nodes, n * M + i, bad) >= 0;
        for (int32_t d = col0 + lane; d < col0 + cols && d < dim; d += kWave) {
            float acc = 0.f;
            const int64_t lo = i - walks.ctx + 1 > 0 ? i - walks.ctx + 1 : 0;
            const int64_t hi = i + walks.ctx - 1 < M - 1 ? i + walks.ctx - 1 : M - 1;
            for (int64_t o = lo; own && o <= hi; ++o) {
                const int64_t v = node_at(walks.nodes, n * M + o, bad);
                const int64_t j = i < o ? i : o;
                if (v < 0 || o == i || j >= walks.windows()) continue;
                acc += band_entry(grad, walks, n, i, o) * E::load(weight[v * row_stride + d]);
            }
            rows[(n * M + i) * dim + d] = acc;
        }
    }
}

// One wavefront: 16 places of a walk, 16 * kPer columns.  The band's entries
// are the first operand, loaded where a lane needs them (lane % 16 the place,
// lane / 16 one of the four other places of a step); the rows the second: lane
// (k, c) holds values 4 c .. 4 c + 3 of place k (and of 16-bit rows 64 + those),
// so that instruction q's columns are the values of index q of every pack, and a
// lane's results are four consecutive values of four places again: stores of
// whole lines.  In float32 throughout: a 16-bit band would round the scores'
// gradients.
//
// Zeros outside the band meet every row of the step, and 0 * inf is NaN: where
// a result is not finite, the tile is done again by the band's products alone.
//
// kRow says how rows are loaded: kWhole, in aligned packs, and dim is a multiple
// of the block's columns; kAligned, in aligned packs that fill the rows;
// kMasked, any.  The first two load without a branch: of places without a node
// the table's first row, of columns past the last the first; their entries are
// 0, or their results not stored.
//
// Bound by the stores (five sixths of what it moves) with the vector units half
// busy beside them: 65,536 walks of 81 nodes, 128 bfloat16, context 10, 4.1 GB in
// 1,050 us (a copy of as many bytes: 850).  One place a wavefront and one column a lane took 15,600.
enum class RowLoad { kWhole, kAligned, kMasked };

template <typename E, RowLoad kRow, bool kStreamed>
__global__ __launch_bounds__(kBlock) void window_rows_grad_kernel(
    const float* __restrict__ grad, const typename E::S* __restrict__ weight, int64_t row_stride,
    int32_t dim, int width, Walks walks, int64_t tiles, float* __restrict__ rows) {
    constexpr int kPer = Matrix<E>::kPer;
    constexpr int kCols = kTileRows * kPer;
    constexpr int kParts = kPer / 4;  // packs of four values
    constexpr int kAhead = 2;         // steps of four places whose loads fly together (4: 1,090 us)
    const int lane = threadIdx.x % kWave;
    const int part = lane / kTileRows, c = lane % kTileRows;
    const int32_t M = walks.walk_nodes, C = walks.ctx;
    const int32_t reach = C - 1;
    const int32_t W = static_cast<int32_t>(walks.windows());
    const int32_t col0 = blockIdx.y * kCols;
    int32_t col[kParts];
#pragma unroll
    for (int h = 0; h < kParts; ++h) col[h] = col0 + h * 4 * kTileRows + c * 4;
    struct Steps {
        Pack<typename E::S, 4> x[kAhead][kParts];
        float a[kAhead];
    };
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave;
         u < walks.num_walks * tiles; u += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t n = u / tiles;
        const int32_t i0 = static_cast<int32_t>(u - n * tiles) * kTileRows;
        // places [from, to) meet the tile's: 16 + 2 * 31 + 3 at most
        const int32_t from = __builtin_amdgcn_readfirstlane(i0 > reach ? (i0 - reach) / 4 * 4 : 0);
        const int32_t span = __builtin_amdgcn_readfirstlane(
            (M - i0 > kTileRows + reach ? i0 + kTileRows + reach : M) - from);
        int32_t node[2];  // of places from + lane, from + 64 + lane
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bool bad = false;
            const int32_t o = h * kWave + lane;
            node[h] = o < span
                          ? static_cast<int32_t>(node_at(walks.nodes, n * M + from + o, bad))
                          : -1;
        }
        // by all lanes: of place from + o, o < 128
        const auto node_of = [&](int32_t o) {
            const int32_t near = __shfl(node[0], o & (kWave - 1), kWave);
            const int32_t far = __shfl(node[1], o & (kWave - 1), kWave);
            return o < kWave ? near : far;
        };
        // places from here on as their distance to `from`
        const int32_t i = i0 - from + c;  // the lane's in the first operand
        const int32_t w = W - from;       // windows start before this one
        const bool own = node_of(i) >= 0;
        // entry (j, j + k) of the band is at band[j * (C - 1) + k]
        const float* band = grad + (n * W + from) * (C - 1) - 1;
        const auto load = [&](Steps& s, int32_t o0) {
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int32_t o = o0 + 4 * q + part;
                const int32_t v = node_of(o);  // -1 from `span` on
                const int32_t j = i < o ? i : o, k = i < o ? o - i : i - o;
                const bool pair = own && v >= 0 && k >= 1 && k < C && j < w;
                s.a[q] = pair ? band[static_cast<uint32_t>(j * (C - 1) + k)] : 0.f;
                const typename E::S* row = weight + static_cast<int64_t>(v < 0 ? 0 : v) * row_stride;
#pragma unroll
                for (int h = 0; h < kParts; ++h)
                    if (kRow == RowLoad::kMasked)
                        s.x[q][h] = load_values<E, 4>(row, col[h], v < 0 ? 0 : dim, width);
                    else
                        s.x[q][h] = *reinterpret_cast<const Pack<typename E::S, 4>*>(
                            row + (kRow == RowLoad::kWhole || col[h] < dim ? col[h] : 0));
            }
        };
        f32x4 acc[kPer];
#pragma unroll
        for (int q = 0; q < kPer; ++q) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
        Steps s;
        load(s, 0);
        for (int32_t o0 = 0; o0 < span; o0 += 4 * kAhead) {
            Steps next;
            if (o0 + 4 * kAhead < span) load(next, o0 + 4 * kAhead);
#pragma unroll
            for (int q = 0; q < kAhead; ++q)
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                        s.a[q], E::load(s.x[q][e / 4].v[e % 4]), acc[e], 0, 0, 0);
            s = next;
        }
        float odd = 0.f;  // NaN if a result is not finite
#pragma unroll
        for (int q = 0; q < kPer; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) odd = __builtin_fmaf(acc[q][r], 0.f, odd);
        if (__ballot(odd != 0.f)) {
            band_rows<E>(grad, weight, row_stride, dim, walks, n, i0, col0, kCols, rows);
            continue;
        }
        float* first = rows + (n * M + i0 + part * 4) * dim;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (i0 + part * 4 + r >= M) continue;
#pragma unroll
            for (int h = 0; h < kParts; ++h) {
                float* to = first + r * dim + col[h];
                if (kRow != RowLoad::kMasked || dim % 4 == 0) {
                    const f32x4 x = {acc[4 * h][r], acc[4 * h + 1][r], acc[4 * h + 2][r],
                                     acc[4 * h + 3][r]};
                    if (kRow != RowLoad::kWhole && col[h] >= dim) continue;
                    if constexpr (kStreamed)
                        __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(to));
                    else
                        *reinterpret_cast<f32x4*>(to) = x;
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (col[h] + q < dim) to[q] = acc[4 * h + q][r];
                }
            }
        }
    }
}

// Walks of one window (windows made elsewhere): the first row's gradient is a
// sum over the others, each of theirs the first row times a number.  Nothing for
// the matrix unit to share: a group of 2^log lanes a walk, a pack of N columns
// each, kBatch rows in flight.  Bound by the rows' stream: 37,700 windows of 10
// nodes, 100 float32 (151 MB read, 151 written) 61 us, 96 in tiles of 16 places;
// whole gradients of 8 to 200,000 such walks of 2 to 32 nodes take 1 to 1 / 1.95
// of the time.
template <typename E, int N, bool kStreamed>
__global__ __launch_bounds__(kBlock) void first_rows_grad_kernel(
    const float* __restrict__ grad, const typename E::S* __restrict__ weight, int64_t row_stride,
    int32_t dim, Walks walks, int log, float* __restrict__ rows) {
    using S = typename E::S;
    constexpr int kBatch = 8;
    const int32_t col = ((blockIdx.y << log) + (threadIdx.x & ((1 << log) - 1))) * N;
    const int32_t M = walks.walk_nodes;
    if (col >= dim) return;
    const auto put = [](float* to, const float (&x)[N]) {
        Pack<float, N> p;
#pragma unroll
        for (int q = 0; q < N; ++q) p.v[q] = x[q];
        if constexpr (kStreamed) stream_pack(to, p);
        else *reinterpret_cast<Pack<float, N>*>(to) = p;
    };
    const int64_t groups = static_cast<int64_t>(gridDim.x) * (kBlock >> log);
    for (int64_t n = (blockIdx.x * static_cast<int64_t>(kBlock) + threadIdx.x) >> log;
         n < walks.num_walks; n += groups) {
        bool bad = false;
        const int64_t own = node_at(walks.nodes, n * M, bad);
        float x0[N], sum[N] = {};
        load_pack<E, N>(x0, weight + (own < 0 ? 0 : own) * row_stride + col);
        float* to = rows + n * M * dim + col;
        for (int32_t k0 = 1; k0 < M; k0 += kBatch) {
            int64_t v[kBatch];
            float c[kBatch];
            Pack<S, N> x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int32_t k = k0 + u < M ? k0 + u : M - 1;
                v[u] = node_at(walks.nodes, n * M + k, bad);
                c[u] = grad[n * (M - 1) + k - 1];
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                x[u] = *reinterpret_cast<const Pack<S, N>*>(weight + (v[u] < 0 ? 0 : v[u]) * row_stride +
                                                            col);
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const bool pair = own >= 0 && v[u] >= 0 && k0 + u < M;
                float y[N];
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const float a = c[u] * E::load(x[u].v[q]), b = c[u] * x0[q];
                    sum[q] += pair ? a : 0.f;
                    y[q] = pair ? b : 0.f;
                }
                if (k0 + u < M) put(to + static_cast<int64_t>(k0 + u) * dim, y);
            }
        }
        put(to, sum);
    }
}

// ------------------------------------------------------------- host side

int wave_grid(int64_t waves, unsigned& grid) {
    DeviceInfo info;
    if (int rc = device_info(info)) return rc;
    int64_t blocks = (waves + kWaves - 1) / kWaves;
    if (blocks > info.cus * 64) blocks = info.cus * 64;
    grid = static_cast<unsigned>(blocks < 1 ? 1 : blocks);
    return MLXC_OK;
}

template <typename E>
int table_width(const Table& table) {
    return pack_width(table.p, table.dim, table.row_stride, sizeof(typename E::S), Matrix<E>::kPer);
}

// Parts of a walk: one wavefront a walk where that fills the device, else its
// row tiles apart.
int split_walks(const Walks& walks, Split& split) {
    DeviceInfo info;
    if (int rc = device_info(info)) return rc;
    const int64_t row_tiles = (walks.windows() + kTileRows - 1) / kTileRows;
    const int64_t want = static_cast<int64_t>(info.cus) * 32;  // wavefronts
    int64_t parts = (want + walks.num_walks - 1) / walks.num_walks;
    if (parts > row_tiles) parts = row_tiles;
    split.per = static_cast<int32_t>((row_tiles + parts - 1) / parts);
    split.parts = static_cast<int32_t>((row_tiles + split.per - 1) / split.per);
    return MLXC_OK;
}

template <typename E, int kSteps, int kAhead, bool kLong>
int scores_launch(const Table& table, const Walks& walks, float scale, float* scores,
                  int64_t* status, hipStream_t stream) {
    Split split;
    unsigned grid;
    if (int rc = split_walks(walks, split)) return rc;
    if (int rc = wave_grid(walks.num_walks * split.parts, grid)) return rc;
    const int width = table_width<E>(table);
    const bool aligned = width == Matrix<E>::kPer && table.num_rows > 0;
    const auto kernel = [aligned] {
        if constexpr (kLong)
            return aligned ? window_scores_long_kernel<E, kSteps, kAhead, true>
                           : window_scores_long_kernel<E, kSteps, kAhead, false>;
        else
            return aligned ? window_scores_kernel<E, kSteps, kAhead, true>
                           : window_scores_kernel<E, kSteps, kAhead, false>;
    }();
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kBlock), 0, stream,
                       static_cast<const typename E::S*>(table.p), table.row_stride, table.dim,
                       width, walks, split, scale, scores, status);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E, int kAhead>
int scores_steps(const Table& table, const Walks& walks, float scale, float* scores,
                 int64_t* status, hipStream_t stream) {
    constexpr int step = Matrix<E>::kStep;
    if (table.dim <= step)
        return scores_launch<E, 1, kAhead, false>(table, walks, scale, scores, status, stream);
    if (table.dim <= 2 * step)
        return scores_launch<E, 2, kAhead, false>(table, walks, scale, scores, status, stream);
    if (table.dim <= 4 * step)
        return scores_launch<E, 4, kAhead, false>(table, walks, scale, scores, status, stream);
    if (table.dim <= 8 * step)
        return scores_launch<E, 8, kAhead, false>(table, walks, scale, scores, status, stream);
    return scores_launch<E, 4, kAhead, true>(table, walks, scale, scores, status, stream);
}

template <typename E>
int scores_typed(const Table& table, const Walks& walks, float scale, float* scores,
                 int64_t* status, hipStream_t stream) {
    // places after a row tile that its last row's pairs reach, in tiles
    if (walks.ctx - 1 <= kTileRows)
        return scores_steps<E, 1>(table, walks, scale, scores, status, stream);
    return scores_steps<E, 2>(table, walks, scale, scores, status, stream);
}

template <typename E, int N>
int first_rows_launch(const float* grad, const Table& table, const Walks& walks, float* rows,
                      bool streamed, hipStream_t stream) {
    int log = 0;
    while (log < 6 && (N << log) < table.dim) ++log;
    const int32_t cols = N << log;
    unsigned grid;
    if (int rc = wave_grid((walks.num_walks << log) / kWave + 1, grid)) return rc;
    auto* kernel = streamed ? first_rows_grad_kernel<E, N, true> : first_rows_grad_kernel<E, N, false>;
    hipLaunchKernelGGL(kernel, dim3(grid, (table.dim + cols - 1) / cols), dim3(kBlock), 0, stream,
                       grad, static_cast<const typename E::S*>(table.p), table.row_stride, table.dim,
                       walks, log, rows);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

template <typename E>
int rows_grad_typed(const float* grad, const Table& table, const Walks& walks, float* rows,
                    hipStream_t stream) {
    constexpr int cols = kTileRows * Matrix<E>::kPer;
    const int64_t tiles = (walks.walk_nodes + kTileRows - 1) / kTileRows;
    unsigned grid;
    if (int rc = wave_grid(walks.num_walks * tiles, grid)) return rc;
    const int width = table_width<E>(table);
    // Rows that the caches cannot hold until they are added up are streamed past
    // them: 5.3 M rows of 128 1,085 -> 1,043 us, and their sums 633 -> 607 (377,000 of 100,
    // 151 MB: 102 -> 89, but the sums 47 -> 63).
    const bool streamed = static_cast<size_t>(walks.count()) * table.dim * sizeof(float) >
                          (size_t{256} << 20);
    if (walks.windows() == 1) {
        if (width >= 4) return first_rows_launch<E, 4>(grad, table, walks, rows, streamed, stream);
        if (width == 2) return first_rows_launch<E, 2>(grad, table, walks, rows, streamed, stream);
        return first_rows_launch<E, 1>(grad, table, walks, rows, streamed, stream);
    }
    const bool whole = table.dim % cols == 0;
    auto* kernel =
        width < 4 ? window_rows_grad_kernel<E, RowLoad::kMasked, false>
        : whole   ? streamed ? window_rows_grad_kernel<E, RowLoad::kWhole, true>
                             : window_rows_grad_kernel<E, RowLoad::kWhole, false>
        : streamed ? window_rows_grad_kernel<E, RowLoad::kAligned, true>
                   : window_rows_grad_kernel<E, RowLoad::kAligned, false>;
    hipLaunchKernelGGL(kernel, dim3(grid, (table.dim + cols - 1) / cols),
                       dim3(kBlock), 0, stream, grad, static_cast<const typename E::S*>(table.p),
                       table.row_stride, table.dim, width, walks, tiles, rows);
    MLXC_HIP_TRY(hipGetLastError());
    return MLXC_OK;
}

__global__ void clear_status_kernel(int64_t* status) {
    if (threadIdx.x == 0) *status = 0;
}

}  // namespace

int launch_window_scores(const Table& table, const Walks& walks, float scale, float* scores,
                         int64_t* status, hipStream_t stream) {
    if (status) {
        hipLaunchKernelGGL(clear_status_kernel, dim3(1), dim3(kWave), 0, stream, status);
        MLXC_HIP_TRY(hipGetLastError());
    }
    if (walks.num_walks == 0) return MLXC_OK;
    if (table.dtype == MLXC_FLOAT32)
        return scores_typed<F32>(table, walks, scale, scores, status, stream);
    if (table.dtype == MLXC_BFLOAT16)
        return scores_typed<BF16>(table, walks, scale, scores, status, stream);
    return scores_typed<F16>(table, walks, scale, scores, status, stream);
}

int launch_window_rows_grad(const float* grad, const Table& table, const Walks& walks, float* rows,
                            hipStream_t stream) {
    // a table without rows: no place has a node, nor a gradient that is read
    if (walks.num_walks == 0 || table.num_rows == 0) return MLXC_OK;
    if (table.dtype == MLXC_FLOAT32) return rows_grad_typed<F32>(grad, table, walks, rows, stream);
    if (table.dtype == MLXC_BFLOAT16) return rows_grad_typed<BF16>(grad, table, walks, rows, stream);
    return rows_grad_typed<F16>(grad, table, walks, rows, stream);
}

}  // namespace mlxc
