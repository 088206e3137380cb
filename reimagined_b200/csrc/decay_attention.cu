// Linear attention with a constant decay for each head: S <- exp(log_decay) S + v k^T, o = scale S q.
//
//   decay_step_kernel        up to four tokens, everything in one launch (heads of a multiple of four)
//   decay_scan_kernel        the recurrence token by token, any size, between (head_rotation.cu), which norms and turns queries and keys, and
//   decay_finish_kernel      head norm and output gate
//   decay_starts_kernel      long scans of few heads: the states before segments of the tokens, which are then scanned side by side
// Prompts in bf16 go by chunks (decay_chunk.cu).
//
// A slow decay enters as S + (exp(log_decay) - 1) S, a fast one as exp(log_decay) S (Decay in decay.cuh).
#include <float.h>

#include <type_traits>

#include "decay.cuh"
#include "flash.cuh"

namespace tbl {
namespace stack {
namespace {

using flash::fma2;
using flash::pair_of;
using flash::unpair;

constexpr int kThreads = 256, kTile = 8, kStepTokens = 4, kMostSegments = 8;

// LK lanes share a value row's keys: lane a holds 4 a + 4 LK j + e for j < C, in pairs of fp32.  A lane holds R rows, a warp 32 / LK times as many.
// Lanes along the keys, so that what all rows multiply with comes out of shared memory in whole lines (eight lanes a row: 328 lines a token for 32
// rows of 90, and they were the bound).
template <int LK, int C, int R>
struct State {
    static constexpr int kKeys = 4 * LK * C, kRows = 32 / LK * R;
    uint64_t s[R][2 * C];

    static __device__ __forceinline__ bool wide(const DecayParams& p) {
        return p.d % 4 == 0 && (reinterpret_cast<uintptr_t>(p.states) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.next) & 15) == 0;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 2 * C; ++j) s[r][j] = 0;
    }
    // rows from `row` on of a head's state in global memory
    __device__ __forceinline__ void load(const DecayParams& p, const float* head, int row, int share) {
        const bool w = wide(p);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float* src = head + static_cast<size_t>(row + r) * p.d;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const int c = 4 * share + 4 * LK * j;
                float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (row + r < p.d) {
                    if (w) {
                        if (c < p.d) f = *reinterpret_cast<const float4*>(src + c);
                    } else {
                        if (c < p.d) f.x = src[c];
                        if (c + 1 < p.d) f.y = src[c + 1];
                        if (c + 2 < p.d) f.z = src[c + 2];
                        if (c + 3 < p.d) f.w = src[c + 3];
                    }
                }
                s[r][2 * j] = pair_of(f.x, f.y);
                s[r][2 * j + 1] = pair_of(f.z, f.w);
            }
        }
    }
    __device__ __forceinline__ void store(const DecayParams& p, float* head, int row, int share) const {
        const bool w = wide(p);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (row + r >= p.d) continue;
            float* dst = head + static_cast<size_t>(row + r) * p.d;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const int c = 4 * share + 4 * LK * j;
                float4 f;
                unpair(s[r][2 * j], f.x, f.y);
                unpair(s[r][2 * j + 1], f.z, f.w);
                if (w) {
                    if (c < p.d) *reinterpret_cast<float4*>(dst + c) = f;
                } else {
                    if (c < p.d) dst[c] = f.x;
                    if (c + 1 < p.d) dst[c + 1] = f.y;
                    if (c + 2 < p.d) dst[c + 2] = f.z;
                    if (c + 3 < p.d) dst[c + 3] = f.w;
                }
            }
        }
    }
    // the same in rows of kKeys, zeros behind a row's numbers
    __device__ __forceinline__ void load_padded(int d, const float* head, int row, int share) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const ulonglong2 f = row + r < d ? *reinterpret_cast<const ulonglong2*>(head + (row + r) * kKeys + 4 * share + 4 * LK * j) : make_ulonglong2(0, 0);
                s[r][2 * j] = f.x;
                s[r][2 * j + 1] = f.y;
            }
    }
    __device__ __forceinline__ void store_padded(int d, float* head, int row, int share) const {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < C; ++j)
                if (row + r < d) *reinterpret_cast<ulonglong2*>(head + (row + r) * kKeys + 4 * share + 4 * LK * j) = make_ulonglong2(s[r][2 * j], s[r][2 * j + 1]);
    }
    // one token: the state, and this lane's share of its rows' outputs; v: the rows' values (R floats, R a multiple of 4 on 16 bytes); m: of Decay, twice
    template <bool SLOW>
    __device__ __forceinline__ void step(uint64_t m, const float* q, const float* k, const float* v, int share, float (&a)[R]) {
        ulonglong2 qq[C], kk[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            qq[j] = *reinterpret_cast<const ulonglong2*>(q + 4 * share + 4 * LK * j);
            kk[j] = *reinterpret_cast<const ulonglong2*>(k + 4 * share + 4 * LK * j);
        }
#pragma unroll
        for (int r = 0; r < R; r += 4) {
            const float4 f = *reinterpret_cast<const float4*>(v + r);
            const float vr[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t vv = pair_of(vr[e], vr[e]);
                uint64_t acc = 0;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    uint64_t &x = s[r + e][2 * j], &y = s[r + e][2 * j + 1];
                    x = fma2(kk[j].x, vv, fma2(m, x, SLOW ? x : 0));
                    y = fma2(kk[j].y, vv, fma2(m, y, SLOW ? y : 0));
                    acc = fma2(qq[j].x, x, acc);
                    acc = fma2(qq[j].y, y, acc);
                }
                float lo, hi;
                unpair(acc, lo, hi);
                a[r + e] = lo + hi;
            }
        }
    }
    // one token's part of a sum, w: its decay
    __device__ __forceinline__ void add(float w, const float* k, const float* v, int share) {
        ulonglong2 kk[C];
#pragma unroll
        for (int j = 0; j < C; ++j) kk[j] = *reinterpret_cast<const ulonglong2*>(k + 4 * share + 4 * LK * j);
#pragma unroll
        for (int r = 0; r < R; r += 4) {
            const float4 f = *reinterpret_cast<const float4*>(v + r);
            const float vr[4] = {f.x * w, f.y * w, f.z * w, f.w * w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t vv = pair_of(vr[e], vr[e]);
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    uint64_t &x = s[r + e][2 * j], &y = s[r + e][2 * j + 1];
                    x = fma2(kk[j].x, vv, x);
                    y = fma2(kk[j].y, vv, y);
                }
            }
        }
    }
    // sums over the lanes of R rows at once: halves of the rows change sides until a lane has one row, rows_at(share)
    static __device__ __forceinline__ float sums(float (&a)[R], int share) {
        int n = R;
#pragma unroll
        for (int o = LK / 2; o; o >>= 1) {
            if (n > 1) {
                n >>= 1;
                const bool upper = (share & o) != 0;
#pragma unroll
                for (int i = 0; i < R / 2; ++i)
                    if (i < n) {
                        const float keep = upper ? a[i + n] : a[i], give = upper ? a[i] : a[i + n];
                        a[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
            } else {
                a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
            }
        }
        return a[0];
    }
    static_assert(R <= LK, "a lane keeps one row");
    static __device__ __forceinline__ int row_at(int share) { return share / (LK / R); }
    static __device__ __forceinline__ bool writes(int share) { return share % (LK / R) == 0; }
};

// norm and gate of a head's output, a warp; x: number lane + 32 i
template <typename T>
__device__ __forceinline__ void finish_head(const DecayParams& p, const float* src, const float* gate, size_t row, int head, int lane) {
    constexpr int kPer = TBL_MAX_ROTATED_DIM / 32;
    float x[kPer], g[kPer], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const bool in = lane + 32 * i < p.d;
        x[i] = in ? src[lane + 32 * i] : 0.0f;
        g[i] = in && gate ? gate[lane + 32 * i] : 0.0f;
        ss = fmaf(x[i], x[i], ss);
    }
    const float f = p.norm ? 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(p.d) + p.eps) : 1.0f;
    T* out = static_cast<T*>(p.out) + (row * p.H + head) * p.d;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c = lane + 32 * i;
        if (c < p.d) out[c] = from_f<T>(x[i] * f * (p.norm ? __ldg(p.norm + head * p.d + c) : 1.0f) * (gate ? sigmoid_f(g[i]) : 1.0f));
    }
}

// Up to four tokens of a head in one launch (32 heads of 128, four tokens 9.2 us, eight 14.1, the scan of nine 11.0; 16 sequences 21.8, 34.7 and
// 31.7).  A CTA has the whole head: its state comes into shared memory by one bulk copy and goes back by another, so that registers hold a few rows
// at a time and three CTAs of heads of 128 share an SM; while it comes, a warp each norms and turns the tokens' queries and keys.  Bound by the
// state's bytes: the projections are asked for first, or they would queue behind the states of the whole batch (64 sequences of 32 heads of 128: 49.7
// us, 5.5 TB/s; with the state in registers 65 to 79).  The bound on registers is what three CTAs have (left to itself the compiler takes 47 instead
// of 60, with fewer loads on their way: 51).
constexpr size_t kStepRoom = 200 * 1024;
size_t step_smem(int keys, int d, int n_tok) { return sizeof(float) * (static_cast<size_t>(d) * d + static_cast<size_t>(n_tok) * (2 * keys + 3 * d)); }

template <typename T, int V, int LK, int C>
__global__ void __launch_bounds__(kThreads, 3) decay_step_kernel(const DecayParams p) {
    using S = State<LK, C, 4>;
    extern __shared__ __align__(128) float room[];
    __shared__ __align__(8) uint64_t full;
    float *state_s = room, *q_s = state_s + p.d * p.d, *k_s = q_s + p.n_tok * S::kKeys, *v_s = k_s + p.n_tok * S::kKeys, *g_s = v_s + p.n_tok * p.d,
          *o_s = g_s + p.n_tok * p.d;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, share = lane % LK;
    const int head = blockIdx.x % p.H, seq = blockIdx.x / p.H;
    const uint32_t bytes = p.d * p.d * 4;
    pdl_launch_dependents();
    if (tid == 0) {
        mbar_init(&full, 1);
        fence_mbar_init();
    }
    if (p.d != S::kKeys)
        for (int i = tid; i < 2 * p.n_tok * S::kKeys; i += kThreads) q_s[i] = 0.0f;
    pdl_wait();
    const int slot = p.slots[seq];
    const size_t row0 = static_cast<size_t>(seq) * p.n_tok;
    const float* proj = p.proj + row0 * p.ld + head * p.d;
    static_assert(2 * kStepTokens <= kThreads / 32, "a warp for every vector");
    const int vec = warp >> 1, is_k = warp & 1;                  // a warp's: the query or key of a token
    HeadUnits<V, 32> x;
    if (vec < p.n_tok) x.load(p.r, proj + static_cast<size_t>(vec) * p.ld + is_k * p.H * p.d, p.d, lane);
    for (int i = tid; i < 2 * p.n_tok * p.d; i += kThreads) {
        const int is_g = i >= p.n_tok * p.d, e = i - is_g * p.n_tok * p.d;
        if (!is_g || p.g_off >= 0) v_s[i] = proj[static_cast<size_t>(e / p.d) * p.ld + (is_g ? p.g_off : p.v_off) + e % p.d];
    }
    const size_t at = (static_cast<size_t>(slot) * p.H + head) * p.d * p.d;
    const int pos = p.positions[slot];
    if (tid == 0) {
        mbar_arrive_expect_tx(&full, bytes);
        bulk_g2s(state_s, p.states + at, bytes, &full);
        if (p.r.half > 0 && head == 0 && (pos < 0 || pos + p.n_tok > p.r.positions)) atomicOr(p.status, TBL_DEV_CACHE_FULL);
    }
    __syncthreads();
    if (vec < p.n_tok) {
        x.template turn<float>(p.r, is_k ? p.k_norm : p.q_norm, p.eps, p.r.half > 0 ? min(max(pos + vec, 0), p.r.positions - 1) : 0, p.d, lane);
        x.store(p.r, (is_k ? k_s : q_s) + vec * S::kKeys, p.d, lane);
    }
    const Decay decay(p.log_decay[head]);
    const uint64_t m = pair_of(decay.m, decay.m);
    const bool alive = mbar_wait_bounded(&full, 0, p.status);
    __syncthreads();
    // four rows a lane at a time (d is a multiple of four: all there or none)
    auto rows = [&](auto slow, int r0) {
        const int r = r0 + lane / LK * 4;
        const bool in = r < p.d;
        S s;
        float* mine = state_s + (in ? r : 0) * p.d;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const int c = 4 * share + 4 * LK * j;
                const ulonglong2 f = c < p.d ? *reinterpret_cast<const ulonglong2*>(mine + i * p.d + c) : make_ulonglong2(0, 0);
                s.s[i][2 * j] = f.x;
                s.s[i][2 * j + 1] = f.y;
            }
        for (int n = 0; n < p.n_tok; ++n) {
            float a[4];
            s.template step<decltype(slow)::value>(m, q_s + n * S::kKeys, k_s + n * S::kKeys, v_s + n * p.d + (in ? r : 0), share, a);
            const float o = S::sums(a, share);
            if (in && S::writes(share)) o_s[n * p.d + r + S::row_at(share)] = o * p.scale;
        }
        __syncwarp();                                            // (lanes without rows have read others')
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const int c = 4 * share + 4 * LK * j;
                if (in && c < p.d) *reinterpret_cast<ulonglong2*>(mine + i * p.d + c) = make_ulonglong2(s.s[i][2 * j], s.s[i][2 * j + 1]);
            }
    };
    for (int r0 = warp * S::kRows; r0 < p.d; r0 += kThreads / 32 * S::kRows) {
        if (decay.slow) rows(std::true_type{}, r0);
        else rows(std::false_type{}, r0);
    }
    fence_proxy_async();
    __syncthreads();
    if (tid == 0 && alive) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.next + at), "r"(smem_u32(state_s)), "r"(bytes) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    for (int t = warp; t < p.n_tok; t += kThreads / 32) finish_head<T>(p, o_s + t * p.d, p.g_off < 0 ? nullptr : g_s + t * p.d, row0 + t, head, lane);
    if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");       // shared memory has been read
}

__device__ __forceinline__ void copy4(float* dst, const float* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 4 : 0) : "memory");
}

// Any number of tokens: a CTA of four warps has 4 State::kRows rows of a head, and a segment of the tokens.  Their vectors come by tiles of kTile
// ahead of their use, a thread the same columns of every token; two tokens' instructions mix.  Bound by a token's chain (0.2 us) where a block has an
// SM to itself, by fp32 operations and shared memory where several share one (62 % of the issue slots).  SUMS: from an empty state, and only the
// state after the segment, which is the start of the next (decay_starts_kernel adds what came before).
constexpr int kScanThreads = 128;
template <int LK, int C, int R, bool SUMS>
__global__ void __launch_bounds__(kScanThreads) decay_scan_kernel(const DecayParams p) {
    using S = State<LK, C, R>;
    constexpr int kRows = kScanThreads / 32 * S::kRows, kFirst = SUMS ? S::kKeys : 0, kCols = 2 * S::kKeys + kRows;
    constexpr int kPer = (kCols - kFirst + kScanThreads - 1) / kScanThreads;
    __shared__ __align__(16) float vec_s[2][kTile][kCols];       // queries, keys, values
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, share = lane % LK, first = warp * S::kRows + lane / LK * R;
    const int head = blockIdx.x % p.H, seq = blockIdx.x / p.H, row0 = blockIdx.y * kRows, part = blockIdx.z;
    const int tokens = min(p.segment, p.n_tok - part * p.segment);
    pdl_wait();
    const size_t numbers = static_cast<size_t>(p.d) * p.d, token0 = static_cast<size_t>(seq) * p.n_tok + static_cast<size_t>(part) * p.segment;
    const size_t state = (static_cast<size_t>(p.slots[seq]) * p.H + head) * numbers;
    float* starts = p.starts + (static_cast<size_t>(blockIdx.x) * p.segments + part) * p.d * S::kKeys;
    const float* src[kPer];
    size_t stride[kPer];
    bool in[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c = kFirst + tid + i * kScanThreads, e = c < S::kKeys ? c : c < 2 * S::kKeys ? c - S::kKeys : row0 + c - 2 * S::kKeys;
        in[i] = c < kCols && e < p.d;
        const size_t at = (token0 * p.H + head) * p.d + (in[i] ? e : 0);
        src[i] = c < S::kKeys ? p.q + at : c < 2 * S::kKeys ? p.k + at : p.proj + token0 * p.ld + p.v_off + head * p.d + (in[i] ? e : 0);
        stride[i] = c < 2 * S::kKeys ? static_cast<size_t>(p.H) * p.d : p.ld;
    }
    auto fetch = [&](int t0, int buf) {
        const int n = min(kTile, tokens - t0);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int c = kFirst + tid + i * kScanThreads;
            if (c >= kCols) break;
#pragma unroll
            for (int t = 0; t < kTile; ++t) {
                if (t >= n) break;
                copy4(&vec_s[buf][t][c], src[i], in[i]);
                src[i] += stride[i];
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0, 0);
    S s;
    if constexpr (SUMS) s.clear();
    else if (p.segments > 1) s.load_padded(p.d, starts, row0 + first, share);
    else s.load(p, p.states + state, row0 + first, share);
    const float rate = p.log_decay[head];
    const Decay decay(rate);
    const uint64_t m = pair_of(decay.m, decay.m);
    const int row = row0 + first + S::row_at(share);
    const bool writes = S::writes(share) && row < p.d;
    float* raw = p.raw + (token0 * p.H + head) * p.d + row;
    auto scan = [&](auto slow) {
        for (int t0 = 0, buf = 0; t0 < tokens; t0 += kTile, buf ^= 1) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();                                         // this tile is there, the one before it is no longer read
            if (t0 + kTile < tokens) fetch(t0 + kTile, buf ^ 1);
            const int n = min(kTile, tokens - t0);
            if constexpr (SUMS) {
#pragma unroll 2
                for (int t = 0; t < n; ++t) {
                    const float kept = expf(t0 + t == tokens - 1 ? 0.0f : rate * static_cast<float>(tokens - 1 - t0 - t));       // (a branch: 60 us instead of 58)
                    s.add(kept, vec_s[buf][t] + S::kKeys, vec_s[buf][t] + 2 * S::kKeys + first, share);
                }
                continue;
            }
            auto token = [&](int t, float (&a)[R]) {
                const float* v = vec_s[buf][t];
                s.template step<decltype(slow)::value>(m, v, v + S::kKeys, v + 2 * S::kKeys + first, share, a);
            };
            int t = 0;
            for (; t + 2 <= n; t += 2) {
                float a[R], b[R];
                token(t, a);
                token(t + 1, b);
                const float x = S::sums(a, share), y = S::sums(b, share);
                if (writes) {
                    raw[0] = x * p.scale;
                    raw[static_cast<size_t>(p.H) * p.d] = y * p.scale;
                }
                raw += 2 * static_cast<size_t>(p.H) * p.d;
            }
            if (t < n) {
                float a[R];
                token(t, a);
                const float x = S::sums(a, share);
                if (writes) raw[0] = x * p.scale;
                raw += static_cast<size_t>(p.H) * p.d;
            }
        }
    };
    if (SUMS || decay.slow) scan(std::true_type{});
    else scan(std::false_type{});
    pdl_launch_dependents();
    if constexpr (SUMS) s.store_padded(p.d, starts + p.d * S::kKeys, row0 + first, share);
    else if (part == p.segments - 1) s.store(p, p.next + state, row0 + first, share);
}

// The states before the segments, a thread per number of rows of `keys`: entry s > 0 holds what segment s - 1 adds to an empty state.
__global__ void __launch_bounds__(256) decay_starts_kernel(const DecayParams p, int keys) {
    pdl_launch_dependents();
    pdl_wait();
    const int unit = blockIdx.y, numbers = p.d * keys, i = blockIdx.x * 256 + threadIdx.x, row = i / keys, col = i % keys;
    if (i >= numbers) return;
    const int head = unit % p.H, slot = p.slots[unit / p.H];
    float* at = p.starts + static_cast<size_t>(unit) * p.segments * numbers + i;
    const Decay decay(p.log_decay[head] * static_cast<float>(p.segment));
    float s = col < p.d ? p.states[((static_cast<size_t>(slot) * p.H + head) * p.d + row) * p.d + col] : 0.0f;
    float x[kMostSegments];
#pragma unroll
    for (int k = 1; k < kMostSegments; ++k) x[k] = k < p.segments ? at[static_cast<size_t>(k) * numbers] : 0.0f;
    at[0] = s;
#pragma unroll
    for (int k = 1; k < kMostSegments; ++k)
        if (k < p.segments) {
            s = decay.of(s) + x[k];
            at[static_cast<size_t>(k) * numbers] = s;
        }
}

// A warp per head of a row.
template <typename T>
__global__ void __launch_bounds__(256) decay_finish_kernel(const DecayParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x, head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (head >= p.H) return;
    const float* gate = p.g_off < 0 ? nullptr : p.proj + static_cast<size_t>(row) * p.ld + p.g_off + head * p.d;
    finish_head<T>(p, p.raw + (static_cast<size_t>(row) * p.H + head) * p.d, gate, row, head, threadIdx.x & 31);
}

int keys_of(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }
bool step_supported(const tbl_decay_mixer& m, int n_tok) { return n_tok <= kStepTokens && m.dim % 4 == 0 && step_smem(keys_of(m.dim), m.dim, n_tok) <= kStepRoom; }
template <typename T, int V, int LK, int C>
cudaError_t launch_step_lk(const DecayParams& p, cudaStream_t st) {
    static bool done[64] = {};
    const size_t smem = step_smem(4 * LK * C, p.d, p.n_tok);
    const cudaError_t e = allow_smem(decay_step_kernel<T, V, LK, C>, smem, done);
    return e != cudaSuccess ? e : launch_dependent(decay_step_kernel<T, V, LK, C>, dim3(p.n_seq * p.H), dim3(kThreads), smem, st, p);
}
template <typename T, int V>
cudaError_t launch_step_v(const DecayParams& p, cudaStream_t st) {
    switch (keys_of(p.d)) {
        case 32: return launch_step_lk<T, V, 8, 1>(p, st);
        case 64: return launch_step_lk<T, V, 16, 1>(p, st);
        case 128: return launch_step_lk<T, V, 32, 1>(p, st);
        default: return launch_step_lk<T, V, 32, 2>(p, st);
    }
}
template <typename T>
cudaError_t launch_step(const DecayParams& p, cudaStream_t st) {
    return p.vec ? launch_step_v<T, 4>(p, st) : launch_step_v<T, 1>(p, st);
}

template <int LK, int C, int R>
cudaError_t launch_scan_r(const DecayParams& p, cudaStream_t st) {
    const unsigned units = p.n_seq * p.H, rows = ceil_div(p.d, kScanThreads / 32 * State<LK, C, R>::kRows);
    if (p.n_tok <= kTile) return launch_dependent(decay_scan_kernel<LK, C, R, false>, dim3(units, rows), dim3(kScanThreads), 0, st, p);
    // Behind a kernel of many rows an early launch finds room on few SMs and stays there, several blocks to one (2000 tokens of 8 heads of 128: 263
    // and 119 us, three prompts of 301 tokens, 10 heads of 90, 59 and 54).
    if (p.segments > 1) {
        decay_scan_kernel<LK, C, R, true><<<dim3(units, rows, p.segments - 1), kScanThreads, 0, st>>>(p);
        note_launch();
        constexpr int keys = State<LK, C, R>::kKeys;
        const cudaError_t e = launch_dependent(decay_starts_kernel, dim3(ceil_div(p.d * keys, 256), units), dim3(256), 0, st, p, keys);
        if (e != cudaSuccess) return e;
    }
    decay_scan_kernel<LK, C, R, false><<<dim3(units, rows, p.segments), kScanThreads, 0, st>>>(p);
    note_launch();
    return cudaGetLastError();
}
// rows of a lane: twice as many once that leaves every SM two blocks
int scan_rows(long long units, int d) { return keys_of(d) == 128 && units >= 2 * kNumSm ? 16 : keys_of(d) <= 64 ? 4 : 8; }
cudaError_t launch_scan(const DecayParams& p, cudaStream_t st) {
    switch (keys_of(p.d)) {
        case 32: return launch_scan_r<8, 1, 4>(p, st);
        case 64: return launch_scan_r<16, 1, 4>(p, st);
        case 128: return scan_rows(static_cast<long long>(p.n_seq) * p.H, p.d) == 16 ? launch_scan_r<32, 1, 16>(p, st) : launch_scan_r<32, 1, 8>(p, st);
        default: return launch_scan_r<32, 2, 8>(p, st);
    }
}
// Segments of a scan: a block takes its tokens one after the other, so few heads leave the GPU empty; with segments the tokens are read twice, by
// more blocks.  Times in us: a token 0.2 where a block has an SM to itself, 0.1 for each block where they share one, sums alone half of that; the
// other two launches 9.5.  Fewest of that wins (fp32, without and with: three prompts of 301 tokens, 10 heads of 90, 75 and 54; 32 heads of 128, 64
// tokens 22 and 28, 300 tokens 72 and 64; 8 heads, 2000 tokens 405 and 119).
int scan_segments(int heads, int d, int n_seq, int n_tok) {
    const long long units = static_cast<long long>(n_seq) * heads;
    const int keys = keys_of(d), lanes = keys <= 32 ? 8 : keys <= 64 ? 16 : 32;
    const double share = static_cast<double>(units) * ceil_div(d, kScanThreads / 32 * (32 / lanes) * scan_rows(units, d)) / kNumSm;       // blocks to an SM
    auto token = [&](int s) { return (0.1 * share * s > 0.2 ? 0.1 * share * s : 0.2) / s; };
    int best = 2;
    for (int s = 3; s <= kMostSegments; ++s)
        if (token(s) <= 1.01 * token(best)) best = s;
    return units <= 65535 && 9.5 + 1.5 * n_tok * token(best) < n_tok * token(1) ? best : 1;
}

enum Route { kAuto = 0, kScan = 1, kChunk = 2 };
// Tokens from which the chunks are faster than the scan: few heads leave both waiting for one chain (32 heads of 128, scan and chunks: 48 tokens 19
// and 23 us, 64 27 and 24; 256 heads: 48 tokens 55 and 50).
int chunk_min_tokens(long long units) { return units >= kNumSm ? 48 : 64; }

struct Plan {
    int route, whole, segments;  // whole: the scan of a few tokens in one launch
    size_t q, k, raw, starts, chunk, bytes;
};

Plan make_plan(const tbl_decay_mixer& m, int precision, int route, int n_seq, int n_tok) {
    Plan w{};
    const long long units = static_cast<long long>(n_seq) * m.heads;
    w.route = route != kAuto ? route : precision == TBL_BF16 && n_tok >= chunk_min_tokens(units) && decay_chunk_supported(m) && units <= 65535 ? kChunk : kScan;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += round_up(bytes, 256); return at; };
    w.whole = w.route == kScan && step_supported(m, n_tok);
    const size_t numbers = w.route == kScan && !w.whole ? static_cast<size_t>(n_seq) * n_tok * m.heads * m.dim : 0;
    w.q = take(4 * numbers);
    w.k = take(4 * numbers);
    w.raw = take(4 * numbers);
    w.segments = numbers ? scan_segments(m.heads, m.dim, n_seq, n_tok) : 1;
    w.starts = take(w.segments > 1 ? sizeof(float) * n_seq * m.heads * w.segments * m.dim * keys_of(m.dim) : 0);
    w.chunk = take(w.route == kChunk ? decay_chunk_workspace(m, n_seq, n_tok) : 0);
    w.bytes = off > 0 ? off : 256;
    return w;
}

// Bytes of a route.  Without one (0), room for whatever as many tokens or fewer take: a host may ask once for its longest portion.
size_t bytes_of(const tbl_decay_mixer& m, int precision, int route, int n_seq, int n_tok) {
    const Plan w = make_plan(m, precision, route, n_seq, n_tok);
    if (route != kAuto || w.route != kChunk) return w.bytes;
    const size_t scan = make_plan(m, precision, kScan, n_seq, chunk_min_tokens(static_cast<long long>(n_seq) * m.heads) - 1).bytes;
    return w.bytes > scan ? w.bytes : scan;
}

}  // namespace

int check_decay(const tbl_decay_mixer& m, int width) {
    if (m.heads <= 0 || m.heads > 65535) return TBL_ERR_SHAPE;
    const int rc = check_rotation(m.rotation, m.dim);
    if (rc != TBL_OK) return rc;
    if (!m.log_decay || (m.gated != 0 && m.gated != 1)) return TBL_ERR_INVALID_ARG;
    if (!(fabsf(m.scale) <= FLT_MAX)) return TBL_ERR_SCALE;
    if (m.in.inputs != width || m.in.outputs != static_cast<long long>(3 + m.gated) * m.heads * m.dim || m.out.inputs != m.heads * m.dim || m.out.outputs != width)
        return TBL_ERR_SHAPE;
    return m.in.weight && m.out.weight ? TBL_OK : TBL_ERR_INVALID_ARG;
}

size_t decay_slot_bytes(const tbl_decay_mixer& m) { return sizeof(float) * static_cast<size_t>(m.heads) * m.dim * m.dim; }

size_t decay_workspace(const tbl_decay_mixer& m, int precision, int n_seq, int n_tok) { return bytes_of(m, precision, kAuto, n_seq, n_tok); }

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
    if (w.whole) return (precision == TBL_BF16 ? launch_step<bf16>(p, st) : launch_step<float>(p, st)) == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
    float *q = reinterpret_cast<float*>(base + w.q), *k = reinterpret_cast<float*>(base + w.k);
    p.q = q; p.k = k; p.raw = reinterpret_cast<float*>(base + w.raw);
    p.starts = reinterpret_cast<float*>(base + w.starts);
    p.segment = ceil_div(n_tok, w.segments);
    p.segments = ceil_div(n_tok, p.segment);
    const RotationCall c{proj, p.ld, m.heads, m.heads, m.dim, slots, positions, n_seq, n_tok, eps, q, k, nullptr, 0};
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
    return bytes_of(*mixer, precision, route, n_seq, n_tok);
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
