// Linear attention with a constant decay for each head: S <- exp(log_decay) S + v k^T, o = scale S q.
//
//   (head_rotation.cu)       queries and keys, normed and turned
//   decay_scan_kernel        the recurrence token by token, fp32: any size, single tokens and short portions
//   decay_finish_kernel      head norm and output gate
// Prompts in bf16 go by chunks (decay_chunk.cu).
//
// The decay enters as S + (exp(log_decay) - 1) S: 1 - exp(log_decay) has 24 bits however slow the decay is, whereas a decay rounded to fp32 would be off by 2^-25
// every token, all in one direction.
#include "decay.cuh"

namespace tbl {
namespace stack {
namespace {

constexpr int kScanThreads = 256, kScanTile = 8;

__device__ __forceinline__ void copy4(float* dst, const float* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 4 : 0) : "memory");
}

// Eight lanes share a value row's keys, KP keys each (lane a holds 4 a + 32 j + e); a lane holds R rows, a CTA 32 R.  The tokens' vectors come by tiles of
// kScanTile ahead of their use.
template <int KP, int R>
__global__ void __launch_bounds__(kScanThreads) decay_scan_kernel(const DecayParams p) {
    constexpr int kKeys = 8 * KP, kRows = 32 * R;
    __shared__ __align__(16) float q_s[2][kScanTile][kKeys], k_s[2][kScanTile][kKeys];
    __shared__ float v_s[2][kScanTile][kRows];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, share = lane & 7;
    const int head = blockIdx.x % p.H, seq = blockIdx.x / p.H, row0 = blockIdx.y * kRows;
    pdl_wait();
    const int slot = p.slots[seq], first = warp * 4 * R + (lane >> 3) * R;       // first of this lane's rows within the CTA's
    const size_t state = (static_cast<size_t>(slot) * p.H + head) * p.d * p.d;
    auto fetch = [&](int t0, int buf) {
        const int n = min(kScanTile, p.n_tok - t0);
        for (int i = tid; i < n * (2 * kKeys + kRows); i += kScanThreads) {
            const int t = i / (2 * kKeys + kRows), c = i - t * (2 * kKeys + kRows);
            const size_t row = static_cast<size_t>(seq) * p.n_tok + t0 + t, at = (row * p.H + head) * p.d;
            if (c < kKeys) copy4(&q_s[buf][t][c], p.q + at + (c < p.d ? c : 0), c < p.d);
            else if (c < 2 * kKeys) copy4(&k_s[buf][t][c - kKeys], p.k + at + (c - kKeys < p.d ? c - kKeys : 0), c - kKeys < p.d);
            else {
                const int r = row0 + c - 2 * kKeys;
                copy4(&v_s[buf][t][c - 2 * kKeys], p.proj + row * p.ld + p.v_off + head * p.d + (r < p.d ? r : 0), r < p.d);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0, 0);
    float s[R][KP];
    const bool wide = p.d % 4 == 0 && (reinterpret_cast<uintptr_t>(p.states) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.next) & 15) == 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + first + r;
        const float* src = p.states + state + static_cast<size_t>(row) * p.d;
#pragma unroll
        for (int j = 0; j < KP / 4; ++j) {
            const int c = 4 * share + 32 * j;
            if (wide) {
                const float4 f = row < p.d && c < p.d ? *reinterpret_cast<const float4*>(src + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                s[r][4 * j] = f.x; s[r][4 * j + 1] = f.y; s[r][4 * j + 2] = f.z; s[r][4 * j + 3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][4 * j + e] = row < p.d && c + e < p.d ? src[c + e] : 0.0f;
            }
        }
    }
    const float less = expm1f(p.log_decay[head]);
    for (int t0 = 0, buf = 0; t0 < p.n_tok; t0 += kScanTile, buf ^= 1) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();                                         // this tile is there, the one before it is no longer read
        if (t0 + kScanTile < p.n_tok) fetch(t0 + kScanTile, buf ^ 1);
        const int n = min(kScanTile, p.n_tok - t0);
        for (int t = 0; t < n; ++t) {
            float v[R], a[R];
#pragma unroll
            for (int r = 0; r < R; ++r) { v[r] = v_s[buf][t][first + r]; a[r] = 0.0f; }
#pragma unroll
            for (int j = 0; j < KP / 4; ++j) {
                const float4 q = *reinterpret_cast<const float4*>(&q_s[buf][t][4 * share + 32 * j]);
                const float4 k = *reinterpret_cast<const float4*>(&k_s[buf][t][4 * share + 32 * j]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float* x = &s[r][4 * j];
                    x[0] = fmaf(k.x, v[r], fmaf(less, x[0], x[0])); a[r] = fmaf(q.x, x[0], a[r]);
                    x[1] = fmaf(k.y, v[r], fmaf(less, x[1], x[1])); a[r] = fmaf(q.y, x[1], a[r]);
                    x[2] = fmaf(k.z, v[r], fmaf(less, x[2], x[2])); a[r] = fmaf(q.z, x[2], a[r]);
                    x[3] = fmaf(k.w, v[r], fmaf(less, x[3], x[3])); a[r] = fmaf(q.w, x[3], a[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int o = 4; o; o >>= 1) a[r] += __shfl_xor_sync(0xffffffffu, a[r], o);
                const int row = row0 + first + r;
                if (share == 0 && row < p.d) p.raw[((static_cast<size_t>(seq) * p.n_tok + t0 + t) * p.H + head) * p.d + row] = a[r] * p.scale;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + first + r;
        if (row >= p.d) continue;
        float* dst = p.next + state + static_cast<size_t>(row) * p.d;
#pragma unroll
        for (int j = 0; j < KP / 4; ++j) {
            const int c = 4 * share + 32 * j;
            if (wide) {
                if (c < p.d) *reinterpret_cast<float4*>(dst + c) = make_float4(s[r][4 * j], s[r][4 * j + 1], s[r][4 * j + 2], s[r][4 * j + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < p.d) dst[c + e] = s[r][4 * j + e];
            }
        }
    }
}

// A warp per head of a row.
template <typename T>
__global__ void __launch_bounds__(256) decay_finish_kernel(const DecayParams p) {
    constexpr int kPer = TBL_MAX_ROTATED_DIM / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x, lane = threadIdx.x & 31, head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (head >= p.H) return;
    const float* src = p.raw + (static_cast<size_t>(row) * p.H + head) * p.d;
    const float* gate = p.g_off < 0 ? nullptr : p.proj + static_cast<size_t>(row) * p.ld + p.g_off + head * p.d;
    float x[kPer], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { x[i] = lane + 32 * i < p.d ? src[lane + 32 * i] : 0.0f; ss = fmaf(x[i], x[i], ss); }
    const float f = p.norm ? 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(p.d) + p.eps) : 1.0f;
    T* out = static_cast<T*>(p.out) + (static_cast<size_t>(row) * p.H + head) * p.d;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c = lane + 32 * i;
        if (c < p.d) out[c] = from_f<T>(x[i] * f * (p.norm ? __ldg(p.norm + head * p.d + c) : 1.0f) * (gate ? sigmoid_f(gate[c]) : 1.0f));
    }
}

template <int KP, int R>
cudaError_t launch_scan_r(const DecayParams& p, cudaStream_t st) {
    return launch_dependent(decay_scan_kernel<KP, R>, dim3(p.n_seq * p.H, ceil_div(p.d, 32 * R)), dim3(kScanThreads), 0, st, p);
}
template <int KP, int MOST>
cudaError_t launch_scan_kp(const DecayParams& p, cudaStream_t st) {
    // as many rows to a lane as still leave two CTAs to an SM
    const long long units = static_cast<long long>(p.n_seq) * p.H;
    if (MOST >= 4 && units * ceil_div(p.d, 128) >= 2 * kNumSm) return launch_scan_r<KP, MOST>(p, st);
    if (MOST >= 2 && units * ceil_div(p.d, 64) >= 2 * kNumSm) return launch_scan_r<KP, MOST < 2 ? MOST : 2>(p, st);
    return launch_scan_r<KP, 1>(p, st);
}
cudaError_t launch_scan(const DecayParams& p, cudaStream_t st) {
    if (p.d <= 32) return launch_scan_kp<4, 1>(p, st);
    if (p.d <= 64) return launch_scan_kp<8, 2>(p, st);
    if (p.d <= 128) return launch_scan_kp<16, 4>(p, st);
    return launch_scan_kp<32, 2>(p, st);
}

enum Route { kAuto = 0, kScan = 1, kChunk = 2 };
constexpr int kChunkMinTokens = 48;

struct Plan {
    int route;
    size_t q, k, raw, chunk, bytes;
};

Plan make_plan(const tbl_decay_mixer& m, int precision, int route, int n_seq, int n_tok) {
    Plan w{};
    w.route = route != kAuto ? route : precision == TBL_BF16 && n_tok >= kChunkMinTokens && decay_chunk_supported(m) ? kChunk : kScan;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += round_up(bytes, 256); return at; };
    const size_t numbers = w.route == kScan ? static_cast<size_t>(n_seq) * n_tok * m.heads * m.dim : 0;
    w.q = take(4 * numbers);
    w.k = take(4 * numbers);
    w.raw = take(4 * numbers);
    w.chunk = take(w.route == kChunk ? decay_chunk_workspace(m, n_seq, n_tok) : 0);
    w.bytes = off;
    return w;
}

}  // namespace

int check_decay(const tbl_decay_mixer& m, int width) {
    if (m.heads <= 0 || m.heads > 65535) return TBL_ERR_SHAPE;
    const int rc = check_rotation(m.rotation, m.dim);
    if (rc != TBL_OK) return rc;
    if (!m.log_decay || (m.gated != 0 && m.gated != 1)) return TBL_ERR_INVALID_ARG;
    if (m.in.inputs != width || m.in.outputs != static_cast<long long>(3 + m.gated) * m.heads * m.dim || m.out.inputs != m.heads * m.dim || m.out.outputs != width)
        return TBL_ERR_SHAPE;
    return m.in.weight && m.out.weight ? TBL_OK : TBL_ERR_INVALID_ARG;
}

size_t decay_slot_bytes(const tbl_decay_mixer& m) { return sizeof(float) * static_cast<size_t>(m.heads) * m.dim * m.dim; }

size_t decay_workspace(const tbl_decay_mixer& m, int precision, int n_seq, int n_tok) { return make_plan(m, precision, kAuto, n_seq, n_tok).bytes; }

int launch_decay(const tbl_decay_mixer& m, int precision, int route, float eps, const float* proj, const float* states, float* next, const int32_t* slots,
                 const int32_t* positions, int n_seq, int n_tok, void* out, void* ws, cudaStream_t st) {
    const Plan w = make_plan(m, precision, route, n_seq, n_tok);
    const long long rows = static_cast<long long>(n_seq) * n_tok;
    if (rows > 2147483647LL || static_cast<long long>(n_seq) * m.heads > 2147483647LL) return TBL_ERR_SHAPE;
    uint8_t* base = static_cast<uint8_t*>(ws);
    DecayParams p{};
    p.status = device_status_ptr();
    if (!p.status) return TBL_ERR_CUDA;
    p.proj = proj; p.log_decay = m.log_decay; p.norm = m.norm; p.states = states; p.next = next; p.slots = slots; p.positions = positions; p.out = out;
    p.r = rotation_of(m.rotation); p.q_norm = m.rotation.q_norm; p.k_norm = m.rotation.k_norm;
    p.ld = m.in.outputs; p.H = m.heads; p.d = m.dim; p.v_off = 2 * m.heads * m.dim; p.g_off = m.gated ? 3 * m.heads * m.dim : -1;
    p.n_seq = n_seq; p.n_tok = n_tok; p.scale = m.scale; p.eps = eps; p.vec = vector_heads(m.rotation, m.dim, proj, p.ld);
    if (w.route == kChunk) return launch_decay_chunks(m, p, base + w.chunk, st);
    float *q = reinterpret_cast<float*>(base + w.q), *k = reinterpret_cast<float*>(base + w.k);
    p.q = q; p.k = k; p.raw = reinterpret_cast<float*>(base + w.raw);
    const RotationCall c{proj, p.ld, m.heads, m.heads, m.dim, slots, positions, n_seq, n_tok, eps, q, k};
    const int rc = launch_head_rotation(m.rotation, TBL_F32, c, st);
    if (rc != TBL_OK) return rc;
    if (launch_scan(p, st) != cudaSuccess) return TBL_ERR_CUDA;
    const dim3 grid(static_cast<unsigned>(rows), ceil_div(m.heads, 8));
    return (precision == TBL_BF16 ? launch_dependent(decay_finish_kernel<bf16>, grid, dim3(256), 0, st, p)
                                  : launch_dependent(decay_finish_kernel<float>, grid, dim3(256), 0, st, p)) == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

}  // namespace stack
}  // namespace tbl

using namespace tbl;
using namespace tbl::stack;

extern "C" {

size_t tbl_decay_workspace_bytes(const tbl_decay_mixer* mixer, int precision, int route, int n_seq, int n_tok) {
    if (!mixer || (precision != TBL_F32 && precision != TBL_BF16) || route < kAuto || route > kChunk || n_seq <= 0 || n_tok <= 0 ||
        check_decay(*mixer, mixer->in.inputs) != TBL_OK)
        return 0;
    return make_plan(*mixer, precision, route, n_seq, n_tok).bytes;
}

int tbl_decay_forward(const tbl_decay_mixer* mixer, int precision, int route, float eps, const float* proj_dev, const float* states_dev,
                      float* next_states_dev, const int32_t* slots_dev, const int32_t* positions_dev, int n_seq, int n_tok, void* out_dev,
                      void* workspace_dev, size_t workspace_bytes, void* stream) {
    if (!mixer || !proj_dev || !states_dev || !next_states_dev || !slots_dev || !positions_dev || !out_dev || n_seq <= 0 || n_tok <= 0 ||
        (precision != TBL_F32 && precision != TBL_BF16) || route < kAuto || route > kChunk || !(eps >= 0.0f))
        return TBL_ERR_INVALID_ARG;
    const int rc = check_decay(*mixer, mixer->in.inputs);
    if (rc != TBL_OK) return rc;
    if (route == kChunk && (precision != TBL_BF16 || !decay_chunk_supported(*mixer))) return TBL_ERR_SHAPE;
    if (!workspace_dev || workspace_bytes < tbl_decay_workspace_bytes(mixer, precision, route, n_seq, n_tok)) return TBL_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace_dev) & 255) || !aligned16(out_dev) || (reinterpret_cast<uintptr_t>(proj_dev) & 3) ||
        (reinterpret_cast<uintptr_t>(states_dev) & 15) || (reinterpret_cast<uintptr_t>(next_states_dev) & 15))
        return TBL_ERR_ALIGNMENT;
    return launch_decay(*mixer, precision, route, eps, proj_dev, states_dev, next_states_dev, slots_dev, positions_dev, n_seq, n_tok, out_dev, workspace_dev,
                        static_cast<cudaStream_t>(stream));
}

}  // extern "C"
