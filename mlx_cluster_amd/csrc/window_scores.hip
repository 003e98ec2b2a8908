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
// instructions read: no LDS, no barrier, every wavefront on its own.
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
    static constexpr int kPer = 8, kStep = 32;
    static __device__ __forceinline__ f32x4 mul(const Pack<uint16_t, 8>& a, const Pack<uint16_t, 8>& b,
                                                f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Matrix<F16> {
    static constexpr int kPer = 8, kStep = 32;
    static __device__ __forceinline__ f32x4 mul(const Pack<_Float16, 8>& a, const Pack<_Float16, 8>& b,
                                                f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Matrix<F32> {
    static constexpr int kPer = 4, kStep = 16;
    // one value of each lane an instruction: its four take the step's values
    // in another order, the same in both operands
    static __device__ __forceinline__ f32x4 mul(const Pack<float, 4>& a, const Pack<float, 4>& b,
                                                f32x4 c) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[q], b.v[q], c, 0, 0, 0);
        return c;
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

// Values [from, from + kSteps * kStep) of this lane's row (node, -1: zeros).
template <typename E, int kSteps>
__device__ __forceinline__ void load_fragment(Fragment<E, kSteps>& f,
                                              const typename E::S* __restrict__ weight,
                                              int64_t row_stride, int32_t dim, int width,
                                              int64_t node, int32_t from) {
    const int lane = threadIdx.x % kWave;
    const typename E::S* row = weight + (node < 0 ? 0 : node) * row_stride;
    const int32_t end = node < 0 ? 0 : dim;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
        f.v[s] = load_values<E, Matrix<E>::kPer>(
            row, from + s * Matrix<E>::kStep + lane / kTileRows * Matrix<E>::kPer, end, width);
}

// The node of row 16 * t + lane % 16 of a walk, -1 from M on.
__device__ __forceinline__ int64_t tile_node(const Walks& walks, int64_t n, int64_t t, bool& bad) {
    const int64_t i = t * kTileRows + threadIdx.x % kTileRows;
    return i < walks.walk_nodes ? node_at(walks.nodes, n * walks.walk_nodes + i, bad) : -1;
}

// Scores of the pairs between row tile t (rows) and t + ahead (columns).
__device__ __forceinline__ void store_scores(const f32x4& acc, const Walks& walks, int64_t n,
                                             int64_t t, int ahead, uint32_t rows_valid,
                                             uint32_t cols_valid, float scale,
                                             float* __restrict__ scores) {
    const int lane = threadIdx.x % kWave;
    const int64_t W = walks.windows();
    const int c = lane % kTileRows;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int r = lane / kTileRows * 4 + q;
        const int64_t j = t * kTileRows + r;
        const int k = ahead * kTileRows + c - r;
        if (j >= W || k < 1 || k >= walks.ctx) continue;
        const bool both = (rows_valid >> r) & (cols_valid >> c) & 1;
        scores[(n * W + j) * (walks.ctx - 1) + k - 1] = both ? acc[q] * scale : 0.f;
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
template <typename E, int kSteps, int kAhead>
__global__ __launch_bounds__(kBlock) void window_scores_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, int32_t dim, int width,
    Walks walks, Split split, float scale, float* __restrict__ scores, int64_t* status) {
    const int64_t W = walks.windows();
    const int64_t row_tiles = (W + kTileRows - 1) / kTileRows;
    bool bad = false;
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave;
         u < walks.num_walks * split.parts; u += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t n = u / split.parts;
        const int64_t first = (u - n * split.parts) * split.per;
        const int64_t last = first + split.per < row_tiles ? first + split.per : row_tiles;
        Fragment<E, kSteps> f[kAhead + 1];
        uint32_t valid[kAhead + 1];
#pragma unroll
        for (int a = 0; a <= kAhead; ++a) {
            const int64_t node = tile_node(walks, n, first + a, bad);
            valid[a] = static_cast<uint32_t>(__ballot(node >= 0)) & 0xffffu;
            load_fragment<E, kSteps>(f[a], weight, row_stride, dim, width, node, 0);
        }
        int64_t next_node = tile_node(walks, n, first + kAhead + 1, bad);
        for (int64_t t = first; t < last; ++t) {
            Fragment<E, kSteps> next;
            uint32_t next_valid = 0;
            if (t + 1 < last) {
                next_valid = static_cast<uint32_t>(__ballot(next_node >= 0)) & 0xffffu;
                load_fragment<E, kSteps>(next, weight, row_stride, dim, width, next_node, 0);
                next_node = tile_node(walks, n, t + kAhead + 2, bad);
            }
#pragma unroll
            for (int a = 0; a <= kAhead; ++a) {
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                    acc = Matrix<E>::mul(f[0].v[s], f[a].v[s], acc);
                store_scores(acc, walks, n, t, a, valid[0], valid[a], scale, scores);
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
template <typename E, int kSteps, int kAhead>
__global__ __launch_bounds__(kBlock) void window_scores_long_kernel(
    const typename E::S* __restrict__ weight, int64_t row_stride, int32_t dim, int width,
    Walks walks, Split split, float scale, float* __restrict__ scores, int64_t* status) {
    const int64_t W = walks.windows();
    const int64_t row_tiles = (W + kTileRows - 1) / kTileRows;
    bool bad = false;
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave;
         u < walks.num_walks * split.parts; u += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t n = u / split.parts;
        const int64_t first = (u - n * split.parts) * split.per;
        const int64_t last = first + split.per < row_tiles ? first + split.per : row_tiles;
        for (int64_t t = first; t < last; ++t) {
            int64_t node[kAhead + 1];
            f32x4 acc[kAhead + 1];
#pragma unroll
            for (int a = 0; a <= kAhead; ++a) {
                node[a] = tile_node(walks, n, t + a, bad);
                acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            for (int32_t from = 0; from < dim; from += kSteps * Matrix<E>::kStep) {
                Fragment<E, kSteps> f[kAhead + 1];
#pragma unroll
                for (int a = 0; a <= kAhead; ++a)
                    load_fragment<E, kSteps>(f[a], weight, row_stride, dim, width, node[a], from);
#pragma unroll
                for (int a = 0; a <= kAhead; ++a)
#pragma unroll
                    for (int s = 0; s < kSteps; ++s)
                        acc[a] = Matrix<E>::mul(f[0].v[s], f[a].v[s], acc[a]);
            }
            const uint32_t rows_valid = static_cast<uint32_t>(__ballot(node[0] >= 0)) & 0xffffu;
#pragma unroll
            for (int a = 0; a <= kAhead; ++a)
                store_scores(acc[a], walks, n, t, a, rows_valid,
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
__device__ __noinline__ void band_rows(const float* __restrict__ grad,
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
// (k, c) holds values c * kPer + 0 .. kPer - 1 of place k, so that instruction
// q's columns are the values of index q of every pack, and a lane's results are
// kPer consecutive values of four places again.  In float32 throughout: a
// 16-bit band would round the scores' gradients.
//
// Zeros outside the band meet every row of the step, and 0 * inf is NaN: where
// a result is not finite, the tile is done again by the band's products alone.
//
// kAligned: packs of kPer values lie aligned and fill the rows.  Places without
// a node, and columns past the last, then load the table's first row and
// values, without a branch: their entries are 0, or their results not stored.
template <typename E, bool kAligned>
__global__ __launch_bounds__(kBlock) void window_rows_grad_kernel(
    const float* __restrict__ grad, const typename E::S* __restrict__ weight, int64_t row_stride,
    int32_t dim, int width, Walks walks, int64_t tiles, float* __restrict__ rows) {
    constexpr int kPer = Matrix<E>::kPer;
    constexpr int kCols = kTileRows * kPer;
    constexpr int kAhead = 4;  // steps of four places whose loads fly together
    const int lane = threadIdx.x % kWave;
    const int part = lane / kTileRows, c = lane % kTileRows;
    const int32_t M = walks.walk_nodes, C = walks.ctx;
    const int32_t reach = C - 1;
    const int32_t W = static_cast<int32_t>(walks.windows());
    const int32_t col0 = blockIdx.y * kCols, col = col0 + c * kPer;
    struct Steps {
        Pack<typename E::S, kPer> x[kAhead];
        float a[kAhead];
    };
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kWaves) + threadIdx.x / kWave;
         u < walks.num_walks * tiles; u += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t n = u / tiles;
        const int32_t i0 = static_cast<int32_t>(u - n * tiles) * kTileRows;
        const int32_t from = i0 > reach ? (i0 - reach) / 4 * 4 : 0;
        const int32_t to = M - i0 > kTileRows + reach ? i0 + kTileRows + reach : M;
        // the nodes of places [from, from + 128), two a lane (16 + 2 * 31 + 3
        // places at most)
        int32_t node[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bool bad = false;
            const int32_t o = from + h * kWave + lane;
            node[h] = o < to ? static_cast<int32_t>(node_at(walks.nodes, n * M + o, bad)) : -1;
        }
        const auto node_of = [&](int32_t o) {  // by all lanes; o in [from, from + 128)
            const int32_t at = o - from;
            const int32_t near = __shfl(node[0], at & (kWave - 1), kWave);
            const int32_t far = __shfl(node[1], at & (kWave - 1), kWave);
            return at < kWave ? near : far;
        };
        const int32_t i = i0 + c;  // the lane's place in the first operand
        const bool own = node_of(i) >= 0;
        const float* band = grad + n * W * (C - 1) - 1;
        const auto load = [&](Steps& s, int32_t o0) {
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int32_t o = o0 + 4 * q + part;
                const int32_t v = node_of(o);  // -1 from `to` on
                const int32_t j = i < o ? i : o, k = i < o ? o - i : i - o;
                const bool pair = own && v >= 0 && k >= 1 && k < C && j < W;
                s.a[q] = pair ? band[static_cast<int64_t>(j) * (C - 1) + k] : 0.f;
                const typename E::S* row = weight + static_cast<int64_t>(v < 0 ? 0 : v) * row_stride;
                if (kAligned)
                    s.x[q] = *reinterpret_cast<const Pack<typename E::S, kPer>*>(
                        row + (col < dim ? col : 0));
                else
                    s.x[q] = load_values<E, kPer>(row, col, v < 0 ? 0 : dim, width);
            }
        };
        f32x4 acc[kPer];
#pragma unroll
        for (int q = 0; q < kPer; ++q) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
        Steps s;
        load(s, from);
        for (int32_t o0 = from; o0 < to; o0 += 4 * kAhead) {
            Steps next;
            if (o0 + 4 * kAhead < to) load(next, o0 + 4 * kAhead);
#pragma unroll
            for (int q = 0; q < kAhead; ++q)
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(s.a[q], E::load(s.x[q].v[e]),
                                                                  acc[e], 0, 0, 0);
            s = next;
        }
        float odd = 0.f;  // NaN if a result is not finite
#pragma unroll
        for (int q = 0; q < kPer; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) odd += acc[q][r] * 0.f;
        if (__ballot(odd != 0.f)) {
            band_rows<E>(grad, weight, row_stride, dim, walks, n, i0, col0, kCols, rows);
            continue;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int32_t place = i0 + part * 4 + r;
            if (place >= M) continue;
            float* to_row = rows + (n * M + place) * dim + col;
            if (kAligned || dim % 4 == 0) {
#pragma unroll
                for (int q = 0; q < kPer; q += 4)
                    if (col + q < dim)
                        *reinterpret_cast<f32x4*>(to_row + q) =
                            f32x4{acc[q][r], acc[q + 1][r], acc[q + 2][r], acc[q + 3][r]};
            } else {
#pragma unroll
                for (int q = 0; q < kPer; ++q)
                    if (col + q < dim) to_row[q] = acc[q][r];
            }
        }
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
    auto* kernel = kLong ? window_scores_long_kernel<E, kSteps, kAhead>
                         : window_scores_kernel<E, kSteps, kAhead>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kBlock), 0, stream,
                       static_cast<const typename E::S*>(table.p), table.row_stride, table.dim,
                       table_width<E>(table), walks, split, scale, scores, status);
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

template <typename E>
int rows_grad_typed(const float* grad, const Table& table, const Walks& walks, float* rows,
                    hipStream_t stream) {
    constexpr int cols = kTileRows * Matrix<E>::kPer;
    const int64_t tiles = (walks.walk_nodes + kTileRows - 1) / kTileRows;
    unsigned grid;
    if (int rc = wave_grid(walks.num_walks * tiles, grid)) return rc;
    const int width = table_width<E>(table);
    auto* kernel = width == Matrix<E>::kPer ? window_rows_grad_kernel<E, true>
                                            : window_rows_grad_kernel<E, false>;
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
