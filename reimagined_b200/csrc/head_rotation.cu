// Norm and rotation of query and key heads in one pass over stacked projections: y = x / sqrt(mean x^2 + eps) * w, then pairs of dimensions turn by
// the angle of the row's position.  Bound by memory: every number is read once (4 bytes) and written once.  A CTA takes one row, so that its heads share the row's
// entries of the tables in the first-level cache; a head lies in registers of 8, 16 or 32 lanes between the sum of squares and the stores.
#include <string.h>

#include "head_rotation.cuh"

namespace tbl {
namespace stack {
namespace {

struct RotationParams {
    const float *proj, *q_norm, *k_norm;
    const int32_t *slots, *positions;
    void *q, *k;
    int* status;
    Rotation r;
    int ld, q_heads, heads, dim, n_tok;
    float eps;
};

template <typename T, int V, int LPH>
__global__ void __launch_bounds__(1024) head_rotation_kernel(const RotationParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x, group = threadIdx.x / LPH, groups = blockDim.x / LPH, lane = threadIdx.x % LPH;
    const int pos = p.positions[p.slots[row / p.n_tok]] + row % p.n_tok;
    if (p.r.half > 0 && (pos < 0 || pos >= p.r.positions)) {
        if (threadIdx.x == 0) atomicOr(p.status, TBL_DEV_CACHE_FULL);
        return;
    }
    const float* src = p.proj + static_cast<size_t>(row) * p.ld;
    // whole warps go round together: the sum of squares is exchanged between their lanes
    for (int h0 = 0; h0 < p.heads; h0 += groups) {
        const int h = h0 + group, hc = min(h, p.heads - 1);
        HeadUnits<V, LPH> x;
        x.load(p.r, src + hc * p.dim, p.dim, lane);
        const bool is_q = hc < p.q_heads;
        x.template turn<float>(p.r, is_q ? p.q_norm : p.k_norm, p.eps, pos, p.dim, lane);
        if (h >= p.heads) continue;
        T* dst = is_q ? static_cast<T*>(p.q) + (static_cast<size_t>(row) * p.q_heads + h) * p.dim
                      : static_cast<T*>(p.k) + (static_cast<size_t>(row) * (p.heads - p.q_heads) + h - p.q_heads) * p.dim;
        x.store(p.r, dst, p.dim, lane);
    }
}

template <typename T, int V, int LPH>
cudaError_t launch(const RotationParams& p, int rows, cudaStream_t st) {
    // few rows: all heads at once; many: CTAs of up to 512 threads whose rounds are full
    const int lanes = p.heads * LPH, most = rows < 2 * kNumSm ? 1024 : 512;
    const int rounds = ceil_div(lanes, most), groups = ceil_div(p.heads, rounds);
    const int threads = static_cast<int>(round_up(static_cast<size_t>(groups) * LPH, 32));
    return launch_dependent(head_rotation_kernel<T, V, LPH>, dim3(rows), dim3(threads), 0, st, p);
}

template <typename T>
cudaError_t launch_type(const RotationParams& p, int rows, bool vec, cudaStream_t st) {
    if (!vec) return launch<T, 1, 32>(p, rows, st);
    if (p.dim <= 64) return launch<T, 4, 8>(p, rows, st);
    if (p.dim <= 128) return launch<T, 4, 16>(p, rows, st);
    return launch<T, 4, 32>(p, rows, st);
}

}  // namespace

int launch_head_rotation(const tbl_head_rotation& r, int precision, const RotationCall& c, cudaStream_t st) {
    RotationParams p{};
    p.status = device_status_ptr();
    if (!p.status) return TBL_ERR_CUDA;
    p.proj = c.proj; p.q_norm = r.q_norm; p.k_norm = r.k_norm; p.slots = c.slots; p.positions = c.positions; p.q = c.q; p.k = c.k;
    p.r = rotation_of(r); p.ld = c.ld; p.q_heads = c.q_heads; p.heads = c.q_heads + c.k_heads; p.dim = c.dim; p.n_tok = c.n_tok; p.eps = c.eps;
    const bool vec = vector_heads(r, c.dim, c.proj, c.ld) && aligned16(c.q) && aligned16(c.k);
    const int rows = c.n_seq * c.n_tok;
    return (precision == TBL_BF16 ? launch_type<bf16>(p, rows, vec, st) : launch_type<float>(p, rows, vec, st)) == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
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
    if (reinterpret_cast<uintptr_t>(proj_dev) & 3) return TBL_ERR_ALIGNMENT;
    RotationCall c{proj_dev, ld, q_heads, k_heads, dim, slots_dev, positions_dev, n_seq, n_tok, eps, q_heads > 0 ? q_dev : nullptr, k_heads > 0 ? k_dev : nullptr};
    return launch_head_rotation(*rotation, precision, c, static_cast<cudaStream_t>(stream));
}
