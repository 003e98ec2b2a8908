// Host twins of the training operators (embedding.hip, window_scores.hip,
// preference.hip): the same formulas on the calling thread, with sums in 64
// bits, rounded once where they are stored.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "train_host.h"

namespace mlxc {

namespace {

float half_to_float(uint16_t h) {
    const uint32_t sign = static_cast<uint32_t>(h & 0x8000u) << 16;
    const uint32_t exp = (h >> 10) & 31u, man = h & 1023u;
    float mag;
    if (exp == 31) mag = man ? NAN : INFINITY;
    else if (exp == 0) mag = std::ldexp(static_cast<float>(man), -24);
    else mag = std::ldexp(static_cast<float>(man | 1024u), static_cast<int>(exp) - 25);
    uint32_t bits;
    std::memcpy(&bits, &mag, 4);
    bits |= sign;
    std::memcpy(&mag, &bits, 4);
    return mag;
}

// x rounded to nearest even to `digits` significant bits, with no bit below
// 2^lowest, and to infinity past `limit`.
double round_to(double x, int digits, int lowest, double limit) {
    if (x == 0 || !std::isfinite(x)) return x;
    int e;
    std::frexp(x, &e);  // |x| in [2^(e-1), 2^e)
    const int ulp = std::max(e - digits, lowest);
    const double r = std::ldexp(std::nearbyint(std::ldexp(x, -ulp)), ulp);
    return std::fabs(r) > limit ? std::copysign(INFINITY, x) : r;
}

uint16_t to_half(double x) {
    const uint16_t sign = std::signbit(x) ? 0x8000u : 0u;
    if (std::isnan(x)) return sign | 0x7e00u;
    const double r = std::fabs(round_to(x, 11, -24, 65504.0));
    if (std::isinf(r)) return sign | 0x7c00u;
    if (r < std::ldexp(1.0, -14)) return sign | static_cast<uint16_t>(std::ldexp(r, 24));
    int e;
    std::frexp(r, &e);
    const uint16_t man = static_cast<uint16_t>(std::ldexp(r, 11 - e)) & 1023u;
    return sign | static_cast<uint16_t>((e + 14) << 10) | man;
}

uint16_t to_bfloat(double x) {
    // one rounding: to 8 bits from 64, which the float then holds exactly
    const float f = static_cast<float>(round_to(x, 8, -133, 3.3895313892515355e38));
    uint32_t bits;
    std::memcpy(&bits, &f, 4);
    if (std::isnan(x)) return static_cast<uint16_t>((bits >> 16) | 0x7fc0u);
    return static_cast<uint16_t>(bits >> 16);
}

double load_at(const void* p, int32_t dtype, int64_t i) {
    if (dtype == MLXC_FLOAT32) return static_cast<const float*>(p)[i];
    const uint16_t h = static_cast<const uint16_t*>(p)[i];
    if (dtype == MLXC_FLOAT16) return half_to_float(h);
    const uint32_t bits = static_cast<uint32_t>(h) << 16;
    float f;
    std::memcpy(&f, &bits, 4);
    return f;
}

void store_at(void* p, int32_t dtype, int64_t i, double x) {
    if (dtype == MLXC_FLOAT32) static_cast<float*>(p)[i] = static_cast<float>(x);
    else static_cast<uint16_t*>(p)[i] = dtype == MLXC_FLOAT16 ? to_half(x) : to_bfloat(x);
}

int64_t host_node(const Nodes& n, int64_t i, int64_t& status) {
    const int64_t v = n.wide ? static_cast<const int64_t*>(n.p)[i]
                             : static_cast<int64_t>(static_cast<const int32_t*>(n.p)[i]);
    if (static_cast<uint64_t>(v) < static_cast<uint64_t>(n.num_rows)) return v;
    if (v != -1) status |= MLXC_STATUS_BAD_NODE;
    return -1;
}

std::vector<int64_t> host_nodes(const Nodes& n, int64_t count, int64_t& status) {
    std::vector<int64_t> v(static_cast<size_t>(count));
    for (int64_t i = 0; i < count; ++i) v[i] = host_node(n, i, status);
    return v;
}

// Gradient rows by node: add(i, row) adds place i's row to `row` (dim values).
template <typename Add>
void coalesce(const std::vector<int64_t>& nodes, int64_t num_rows, int32_t dim, float scale,
              const GradOut& out, Add add) {
    const int64_t count = static_cast<int64_t>(nodes.size());
    std::vector<int64_t> order;
    for (int64_t i = 0; i < count; ++i)
        if (nodes[i] >= 0) order.push_back(i);
    std::stable_sort(order.begin(), order.end(),
                     [&](int64_t a, int64_t b) { return nodes[a] < nodes[b]; });
    const int64_t rows = out.ids ? std::min(count, num_rows) : num_rows;
    for (int64_t i = 0; i < rows * dim; ++i) store_at(out.p, out.dtype, i, 0.0);
    if (out.ids) std::fill(out.ids, out.ids + rows, int64_t{-1});
    std::vector<double> row(static_cast<size_t>(dim));
    int64_t u = 0;
    for (size_t b = 0; b < order.size(); ++u) {
        const int64_t node = nodes[order[b]];
        std::fill(row.begin(), row.end(), 0.0);
        for (; b < order.size() && nodes[order[b]] == node; ++b) add(order[b], row.data());
        const int64_t at = out.ids ? u : node;
        if (out.ids) out.ids[u] = node;
        for (int32_t d = 0; d < dim; ++d) store_at(out.p, out.dtype, at * dim + d, row[d] * scale);
    }
}

double softplus(double x) { return std::fmax(x, 0.0) + std::log1p(std::exp(-std::fabs(x))); }

}  // namespace

void host_embedding(const Table& table, const Nodes& nodes, int64_t count, float scale, void* out,
                    int64_t& status) {
    for (int64_t i = 0; i < count; ++i) {
        const int64_t v = host_node(nodes, i, status);
        for (int32_t d = 0; d < table.dim; ++d)
            store_at(out, table.dtype, i * table.dim + d,
                     v < 0 ? 0.0 : load_at(table.p, table.dtype, v * table.row_stride + d) * scale);
    }
}

void host_embedding_grad(const void* rows, int32_t dtype, int32_t dim, const Nodes& nodes,
                         int64_t count, float scale, const GradOut& out, int64_t& status) {
    coalesce(host_nodes(nodes, count, status), nodes.num_rows, dim, scale, out,
             [&](int64_t i, double* row) {
                 for (int32_t d = 0; d < dim; ++d) row[d] += load_at(rows, dtype, i * dim + d);
             });
}

void host_window_scores(const Table& table, const Walks& walks, float scale, float* scores,
                        int64_t& status) {
    const int32_t M = walks.walk_nodes, C = walks.ctx;
    const int64_t W = walks.windows();
    const std::vector<int64_t> nodes = host_nodes(walks.nodes, walks.count(), status);
    for (int64_t n = 0; n < walks.num_walks; ++n)
        for (int64_t j = 0; j < W; ++j)
            for (int32_t k = 1; k < C; ++k) {
                const int64_t u = nodes[n * M + j], v = nodes[n * M + j + k];
                double s = 0;
                if (u >= 0 && v >= 0)
                    for (int32_t d = 0; d < table.dim; ++d)
                        s += load_at(table.p, table.dtype, u * table.row_stride + d) *
                             load_at(table.p, table.dtype, v * table.row_stride + d);
                scores[(n * W + j) * (C - 1) + k - 1] =
                    u >= 0 && v >= 0 ? static_cast<float>(s * scale) : 0.f;
            }
}

void host_window_scores_grad(const float* grad, const Table& table, const Walks& walks, float scale,
                             const GradOut& out, int64_t& status) {
    const int32_t M = walks.walk_nodes, C = walks.ctx;
    const int64_t W = walks.windows();
    const std::vector<int64_t> nodes = host_nodes(walks.nodes, walks.count(), status);
    coalesce(nodes, table.num_rows, table.dim, scale, out, [&](int64_t at, double* row) {
        const int64_t n = at / M, i = at % M;
        const int64_t lo = std::max<int64_t>(0, i - C + 1);
        const int64_t hi = std::min<int64_t>(M - 1, i + C - 1);
        for (int64_t o = lo; o <= hi; ++o) {
            const int64_t j = std::min(i, o), k = std::max(i, o) - j;
            const int64_t v = nodes[n * M + o];
            if (k == 0 || j >= W || v < 0) continue;
            const double c = grad[(n * W + j) * (C - 1) + k - 1];
            for (int32_t d = 0; d < table.dim; ++d)
                row[d] += c * load_at(table.p, table.dtype, v * table.row_stride + d);
        }
    });
}

void host_preference_loss(const PreferenceCall& c, float* loss, float* rewards, float* slopes) {
    double total = 0;
    std::vector<float> own;
    if (!slopes && (c.side[0].grad || c.side[1].grad)) {
        own.resize(static_cast<size_t>(2 * c.pairs));
        slopes = own.data();
    }
    const double share = c.sum || c.pairs == 0 ? 1.0 : 1.0 / static_cast<double>(c.pairs);
    for (int64_t p = 0; p < c.pairs; ++p) {
        double r[2], per[2];
        for (int s = 0; s < 2; ++s) {
            const mlxc_preference_side& x = c.side[s];
            double sum = 0;
            int64_t left = 0;
            for (int64_t t = 0; t < x.length; ++t) {
                const int64_t i = p * x.length + t;
                if (x.mask && !x.mask[i]) continue;
                ++left;
                sum += load_at(x.values, c.dtype, i) -
                       (x.reference ? load_at(x.reference, c.dtype, i) : 0.0);
            }
            per[s] = c.normalize ? 1.0 / static_cast<double>(std::max<int64_t>(left, 1)) : 1.0;
            r[s] = c.beta * sum * per[s];
            if (rewards) rewards[s * c.pairs + p] = static_cast<float>(r[s]);
        }
        const double z = r[0] - r[1];
        double l = 0, dz = 0;
        if (c.smoothing < 1.f) {
            l += (1.0 - c.smoothing) * softplus(-z);
            dz -= (1.0 - c.smoothing) / (1.0 + std::exp(z));
        }
        if (c.smoothing > 0.f) {
            l += c.smoothing * softplus(z);
            dz += c.smoothing / (1.0 + std::exp(-z));
        }
        total += l;
        dz *= c.beta * share;
        if (slopes) {
            slopes[p] = static_cast<float>(dz * per[0]);
            slopes[c.pairs + p] = static_cast<float>(-dz * per[1]);
        }
    }
    *loss = static_cast<float>(total * share);
    host_preference_grad(c, slopes, nullptr);
}

void host_preference_grad(const PreferenceCall& c, const float* slopes, const float* upstream) {
    const double up = upstream ? *upstream : 1.0;
    for (int s = 0; s < 2; ++s) {
        const mlxc_preference_side& x = c.side[s];
        if (!x.grad) continue;
        for (int64_t p = 0; p < c.pairs; ++p)
            for (int64_t t = 0; t < x.length; ++t) {
                const int64_t i = p * x.length + t;
                store_at(x.grad, c.dtype, i,
                         x.mask && !x.mask[i] ? 0.0 : up * slopes[s * c.pairs + p]);
            }
    }
}

}  // namespace mlxc
