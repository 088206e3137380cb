// Norm and rotation of query and key heads in one pass over stacked projections: y = x / sqrt(mean x^2 + eps) * w, then pairs of dimensions turn by
// the angle of the row's position.  Bound by memory: every number is read once (4 bytes) and written once.  A CTA takes a row at a time, so that a thread reads
// the row's angles once for all its heads; a head lies in registers of 8, 16 or 32 lanes between the sum of squares and the stores.
// 8192 rows of 32 + 8 heads of 128, bf16: 50 us for 252 MB, 5.0 TB/s.

#include "head_rotation.cuh"

namespace tbl {
namespace stack {
namespace {

struct RotationParams {
    const float *proj, *q_norm, *k_norm;
    const int32_t *slots, *positions;
    void *q, *k;
    float* q_factor;
    int* status;
    Rotation r;
    int ld, q_heads, heads, dim, n_tok, rows, ldq;
    float eps, per_dim;
};

constexpr int kMostThreads = 256;

// LPH lanes a head, U units a lane.  A thread has the same columns of every head it takes: their places and weights stay in registers, a row's angles
// for all its heads.  HALVES: queries as fp16 under a power of two (RotationCall).
template <typename T, int V, int LPH, int U, bool HALVES, bool EXACT>
__global__ void __launch_bounds__(kMostThreads, V == 4 ? 6 : 4) head_rotation_kernel(const RotationParams p) {
    using Units = HeadUnits<V, LPH>;
    constexpr int kRuns = 2 * U, kNumbers = V * kRuns;
    const int dim = EXACT ? kNumbers * LPH : p.dim, limit = EXACT ? 1 << 30 : p.dim;         // limit: of the columns that are there
    const int group = threadIdx.x / LPH, groups = blockDim.x / LPH, gl = threadIdx.x % LPH;
    // a head's lanes: others of the warp may have heads without a norm
    const uint32_t mates = LPH == 32 ? 0xffffffffu : ((1u << (LPH & 31)) - 1u) << (threadIdx.x % 32 / LPH * LPH);
    int at[kRuns];
#pragma unroll
    for (int u = 0; u < U; ++u) Units::runs(p.r, gl + LPH * u, at[2 * u], at[2 * u + 1]);
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x;
    const int pos = p.positions[p.slots[row / p.n_tok]] + row % p.n_tok;
    const bool outside = p.r.half > 0 && (pos < 0 || pos >= p.r.positions);
    if (outside && threadIdx.x == 0) atomicOr(p.status, TBL_DEV_CACHE_FULL);
    if (outside && !HALVES) return;                          // (a step's rows are undefined then, an operator's stay as they were)
    const int entry = p.r.half > 0 ? min(max(pos, 0), p.r.positions - 1) : 0;
    float c[V * U], sn[V * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int n = V * (gl + LPH * u);
#pragma unroll
        for (int e = 0; e < V; ++e) { c[V * u + e] = 1.0f; sn[V * u + e] = 0.0f; }
        if (n < p.r.half) {
            Units::load_run(p.r.cos + static_cast<size_t>(entry) * p.r.half, n, 1 << 30, c + V * u);
            Units::load_run(p.r.sin + static_cast<size_t>(entry) * p.r.half, n, 1 << 30, sn + V * u);
        }
    }
    const float* src = p.proj + static_cast<size_t>(row) * p.ld;
    // whole warps go round together: sums are exchanged between their lanes
    for (int h = group; h - group < p.heads; h += groups) {
        float x[kNumbers], f = 1.0f;
        const bool is_k = h >= p.q_heads;
        const float *head = src + min(h, p.heads - 1) * dim, *norm = is_k ? p.k_norm : p.q_norm;
#pragma unroll
        for (int u = 0; u < kRuns; ++u) Units::load_run(head, at[u], limit, x + V * u);
        if (norm) {
            float ss = 0.0f, w[kNumbers];
#pragma unroll
            for (int u = 0; u < kRuns; ++u) Units::load_run(norm, at[u], limit, w + V * u);
#pragma unroll
            for (int e = 0; e < kNumbers; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(mates, ss, o);
            f = rsqrtf(fmaf(ss, p.per_dim, p.eps));
#pragma unroll
            for (int e = 0; e < kNumbers; ++e) x[e] *= w[e] * f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) turn_unit<V>(p.r.interleaved, c + V * u, sn + V * u, x + 2 * V * u);
        float back = 1.0f;
        if (HALVES) {
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < kNumbers; ++e) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
            for (int o = LPH / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float power = power_of(most);
            back = inverse_power(power) * kUp;
            if (gl == 0 && h < p.heads) p.q_factor[static_cast<size_t>(row) * p.heads + h] = power * (1.0f / kUp);
        }
        if (h >= p.heads) continue;
        T* dst = HALVES ? static_cast<T*>(p.q) + (static_cast<size_t>(row) * p.heads + h) * p.ldq
                 : is_k ? static_cast<T*>(p.k) + (static_cast<size_t>(row) * (p.heads - p.q_heads) + h - p.q_heads) * dim
                        : static_cast<T*>(p.q) + (static_cast<size_t>(row) * p.q_heads + h) * dim;
#pragma unroll
        for (int u = 0; u < kRuns; ++u) Units::store_run(dst, at[u], HALVES ? p.ldq : limit, x + V * u, back);
    }
}

template <typename T, int V, int LPH, int U, bool HALVES, bool EXACT>
cudaError_t launch(const RotationParams& p, cudaStream_t st) {
    // (a CTA for several rows, its lanes' weights kept in registers: 57 to 65 us for 8192 rows of 40 heads of 128, since fewer loads are on their way)
    const int rounds = ceil_div(p.heads * LPH, kMostThreads), groups = ceil_div(p.heads, rounds);
    const int threads = static_cast<int>(round_up(static_cast<size_t>(groups) * LPH, 32));
    return launch_dependent(head_rotation_kernel<T, V, LPH, U, HALVES, EXACT>, dim3(p.rows), dim3(threads), 0, st, p);
}

template <typename T, bool HALVES>
cudaError_t launch_type(const RotationParams& p, int run, cudaStream_t st) {
    if (run == 1) return launch<T, 1, 32, 4, HALVES, false>(p, st);
    if (run == 2) return p.dim <= 128 ? launch<T, 2, 32, 1, HALVES, false>(p, st) : launch<T, 2, 32, 2, HALVES, false>(p, st);
    if (p.dim <= 64) return p.dim == 64 ? launch<T, 4, 8, 1, HALVES, true>(p, st) : launch<T, 4, 8, 1, HALVES, false>(p, st);
    if (p.dim <= 128) return p.dim == 128 ? launch<T, 4, 16, 1, HALVES, true>(p, st) : launch<T, 4, 16, 1, HALVES, false>(p, st);
    return launch<T, 4, 32, 1, HALVES, false>(p, st);
}

}  // namespace

int launch_head_rotation(const tbl_head_rotation& r, int precision, const RotationCall& c, cudaStream_t st) {
    RotationParams p{};
    p.status = device_status_ptr();
    if (!p.status) return TBL_ERR_CUDA;
    p.proj = c.proj; p.q_norm = r.q_norm; p.k_norm = r.k_norm; p.slots = c.slots; p.positions = c.positions; p.q = c.q; p.k = c.k; p.q_factor = c.q_factor;
    p.r = rotation_of(r); p.ld = c.ld; p.q_heads = c.q_heads; p.heads = c.q_heads + c.k_heads; p.dim = c.dim; p.n_tok = c.n_tok; p.eps = c.eps;
    p.rows = c.n_seq * c.n_tok; p.ldq = c.ldq; p.per_dim = 1.0f / static_cast<float>(c.dim);
    // runs of four or two numbers where everything lies on their bytes
    const int run = vector_heads(r, c.dim, c.proj, c.ld) && aligned16(c.q) && aligned16(c.k) ? 4 : paired_heads(r, c.dim, c.proj, c.ld, c.q, c.k) ? 2 : 1;
    const cudaError_t e = c.q_factor ? launch_type<__half, true>(p, run, st) : precision == TBL_BF16 ? launch_type<bf16, false>(p, run, st)
                                                                                                     : launch_type<float, false>(p, run, st);
    return e == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

}  // namespace stack
}  // namespace tbl

using namespace tbl;
using namespace tbl::stack;

extern "C" int tbl_head_rotation_forward(const tbl_head_rotation* rotation, int precision, float eps, const float* proj_dev, int ld, int q_heads,
                                         int k_heads, int dim, const int32_t* slots_dev, const int32_t* positions_dev, int n_seq, int n_tok,
                                         void* q_dev, void* k_dev, void* stream) {
    if (!rotation || !proj_dev || !slots_dev || !positions_dev || q_heads < 0 || k_heads < 0 || (q_heads > 0 && !q_dev) || (k_heads > 0 && !k_dev) ||
        n_seq <= 0 || n_tok <= 0 || (precision != TBL_F32 && precision != TBL_BF16) || !(eps >= 0.0f))
        return TBL_ERR_INVALID_ARG;
    const int rc = check_rotation(*rotation, dim);
    if (rc != TBL_OK) return rc;
    const long long heads = static_cast<long long>(q_heads) + k_heads;
    if (heads == 0) return TBL_ERR_INVALID_ARG;
    if (heads * dim > ld || static_cast<long long>(n_seq) * n_tok > 2147483647LL) return TBL_ERR_SHAPE;
    const uintptr_t own = precision == TBL_BF16 ? 1 : 3;
    if ((reinterpret_cast<uintptr_t>(proj_dev) & 3) || (q_heads > 0 && (reinterpret_cast<uintptr_t>(q_dev) & own)) ||
        (k_heads > 0 && (reinterpret_cast<uintptr_t>(k_dev) & own)))
        return TBL_ERR_ALIGNMENT;
    const RotationCall c{proj_dev, ld, q_heads, k_heads, dim, slots_dev, positions_dev, n_seq, n_tok, eps,
                         q_heads > 0 ? q_dev : nullptr, k_heads > 0 ? k_dev : nullptr, nullptr, 0};
    return launch_head_rotation(*rotation, precision, c, static_cast<cudaStream_t>(stream));
}
