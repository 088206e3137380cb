// Attention of a few query rows over a long 4-bit cache (decode, short portions): the rows of 4-bit numbers stream through shared memory once per
// block of 8 or 16 query rows that share a key/value head, and become matrix operands in registers.
//
// Code x scale (e2m1 x e4m3: six bits between 2^-10 and 2688) is exact in fp16, so the products are warp-level MMAs (16 x 8 x 16, fp16 operands, fp32
// sums) of exact keys and values; queries are rounded to fp16 under a power of two per head, softmax weights to fp16 (2^-12 each, where the bf16
// result is rounded by 2^-9): the largest weight stands at 2^11, so that one down to 2^-25 of it keeps its bits, 2^-35 is left out.  Scores are made
// as S^T = K Q^T and outputs as O^T = V^T P^T: cached numbers are the A operand, whose 16 x 16 numbers a step cost the fewest MMAs, and the fragments
// of S^T turn into those of P^T by one transposed 8 x 8 move each.
//
// The order of the dimensions inside an MMA is free as long as both operands agree, so a lane takes 16 neighbouring dimensions of a token's key --
// one scale -- for four steps, and eight of a value.  For the values two tokens' codes are brought side by side while they are still 4 bits wide (two
// logic operations for sixteen numbers).  A warp of W works alone on every W-th tile of 32 tokens of the CTA's split: a ring of bulk copies of its
// own, its own maxima, sums and outputs; the warps meet in shared memory at the end, splits of the context in quantized_merge_kernel.
//
// No single pipe bounds it.  A tile of 16 tokens of a head of 128 (2304 bytes, 100 cycles of an SM's share of the memory) costs 64 conversions and
// some 40 logic operations on one pipe (two warps a cycle), 64 multiplications on another, 16 MMAs: some 300 instructions.  One token of 64 sequences
// of 8 heads over 4096: 74 us with the kernel ahead, 4.2 TB/s of 302 MB; of one sequence over 131001 46 us, of which this kernel has 37: 58 % of the
// issue slots, the conversions' pipe 51 %, MMAs 25 %, memory 0.63 of a copy's rate, and warps (sixteen to an SM) that wait as long for their turn as
// for results and for the pipe.
#include <float.h>

#include "attention.cuh"
#include "quantized.cuh"
#include "tc05.cuh"

namespace tbl {
namespace stack {
namespace {

constexpr int kTile = 32;
constexpr float kRescale = 4.0f, kTop = 11.0f;           // a weight stays below 2^15

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// the eight codes of a word as four pairs of halves, times a pair of scales (as one piece of assembly the conversions take their byte of the word by
// themselves)
__device__ __forceinline__ void widen(uint32_t codes, __half2 scale, uint32_t (&out)[4]) {
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\ncvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\ncvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3]) : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&out[i]), scale);
        out[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}
// two e4m3 bytes (the low one first) as halves
__device__ __forceinline__ __half2 scales_of(uint32_t bytes) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(bytes), __NV_E4M3);
    return *reinterpret_cast<const __half2*>(&h);
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) { uint32_t v; asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a)); return v; }
// N words from a place of 4 bytes on, pairs at once where it is one of 8
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&v)[N]) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[i]), "=r"(v[i + 1]) : "r"(a + 4 * i));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lds32(a + 4 * i);
    }
}
__device__ __forceinline__ uint2 lds64(uint32_t a) { uint2 v; asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a)); return v; }

// The token (of 16) that stands in row i of an MMA: with rows of 144 bytes the 16 or 32 lanes that a shared-memory access serves together then hit
// every bank once, for the keys (rows 0 .. 3 and 4 .. 7 of the MMA) as for the values (rows 0, 2, 4, 6 and so on).
__device__ __forceinline__ int token_of(int i) {
    const int r = i & 7;
    return ((r & 1) ? 8 + (((r & 6) + 4) & 7) : r) + (i >> 3);
}

template <int DP, int NT, int W>
struct Layout {
    static constexpr int kStages = W == 4 ? 3 : 2, kRow = (DP + DP / 8 + 15) / 16 * 16, kTileBytes = kTile * kRow, kRing = W * kStages * kTileBytes, kLdo = DP + 4;
    static constexpr size_t kMerge = sizeof(float) * W * 8 * NT * kLdo, kBytes = kRing > kMerge ? kRing : kMerge;
};

// The bound on registers is what shared memory leaves blocks for (left to itself the compiler saves some that bring no further block: 64 sequences
// over 4096 tokens 77 instead of 74 us; five blocks with two stages each 74, six 81). DP: the head size rounded up to 64; NT: blocks of eight query
// rows; W: warps; V: 0, or how the vectors of a whole call (StreamPlan) are read (HeadUnits).
template <int DP, int NT, int W, int V>
__global__ void __launch_bounds__(32 * W, W == 16 || DP > 128 ? 1 : NT == 1 ? 4 : 3) quantized_stream_kernel(const QuantizedParams p) {
    using L = Layout<DP, NT, W>;
    constexpr int kBlocks = DP / 64, kRows = 8 * NT, kThreads = 32 * W, kStages = L::kStages;
    constexpr bool kWhole = V > 0;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float m_s[W][kRows], l_s[W][kRows], top_s[kRows], sum_s[kRows];
    __shared__ __align__(8) uint64_t full[W][kStages];
    __shared__ __align__(16) __half q_s[kWhole ? kRows : 1][kWhole ? DP : 8];
    __shared__ __align__(16) float head_s[kWhole ? (W < 8 ? W : 8) : 1][kWhole ? DP : 4], factor_s[kRows];
    __shared__ __align__(16) uint8_t fresh_s[kWhole ? L::kRow : 16];
    float* o_s = reinterpret_cast<float*>(smem);                 // afterwards: [warp][row][kLdo]
    const int tid = threadIdx.x, warp = tc05::uniform_warp(), lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const int seq = blockIdx.x / p.G, g = blockIdx.x % p.G, first = blockIdx.y * kRows, split = blockIdx.z;
    const int total = p.n_tok * p.group;
    if (lane == 0)
        for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
    fence_mbar_init();
    fence_proxy_async();
    __syncthreads();
    pdl_wait();
    const int slot = p.slots[seq], pos0 = p.positions[slot];
    const int n = min(pos0 + min(total - 1, first + kRows - 1) / p.group + 1, p.capacity);       // tokens the last row sees
    const int per = ((n + p.splits - 1) / p.splits + kTile - 1) / kTile * kTile;
    const int t0 = min(split * per, max(n, 0)), t1 = min(n, t0 + per);
    // the token of a whole call (at pos0, the last one) comes from the projections, not from the cache
    const int fresh = kWhole && quantized_room(p, pos0) ? pos0 : -1, cached = fresh >= 0 ? min(t1, fresh) : t1;
    const uint8_t* cache = quantized_at(p, slot, g, 0);
    uint8_t* ring = smem + warp * kStages * L::kTileBytes;
    auto load_tile = [&](int stage, int t) {                     // rows past the split's end stay whatever shared memory holds: they are masked
        if (t < t1 && tc05::elect_one()) {
            const int rows = min(kTile, cached - t);
            if (!kWhole || rows > 0) {
                mbar_arrive_expect_tx(&full[warp][stage], rows * L::kRow);
                bulk_g2s(ring + stage * L::kTileBytes, cache + static_cast<size_t>(t) * L::kRow, rows * L::kRow, &full[warp][stage]);
            } else {
                mbar_arrive(&full[warp][stage]);
            }
        }
    };
    const int begin = t0 + warp * kTile, step = W * kTile;
#pragma unroll
    for (int s = 0; s < kStages; ++s) load_tile(s, begin + s * step);
    if constexpr (kWhole) {                                      // a warp per head: queries, the key, the value
        constexpr int kHeads = W < 8 ? W : 8;
        const float* src = p.proj + static_cast<size_t>(seq) * p.ld;
        const int at = p.r.half > 0 ? min(max(pos0, 0), p.r.positions - 1) : 0;
        for (int i = tid; i < kRows * DP / 8; i += kThreads) reinterpret_cast<uint4*>(&q_s[0][0])[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (warp < kHeads)
            for (int i = warp; i < p.group + 2; i += kHeads) {
                if (i < 2) {                                     // (these first: they take longer)
                    const bool is_k = i == 0;
                    uint8_t scale;
                    const uint32_t codes = quantize_head<V>(p, src + ((is_k ? p.H : p.H + p.G) + g) * p.d, is_k, at, head_s[warp], lane, scale);
                    put_row(p, fresh_s, is_k, codes, scale, lane);
                    if (fresh >= 0) put_row(p, quantized_at(p, slot, g, fresh), is_k, codes, scale, lane);
                } else {
                    HeadUnits<V, 32> x;
                    float f;
                    x.load(p.r, src + (g * p.group + i - 2) * p.d, p.d, lane);
                    x.template turn<float>(p.r, p.q_norm, p.eps, at, p.d, lane);
                    const float power = query_power(x, f);
                    if (lane == 0) factor_s[i - 2] = power;
                    x.store(p.r, q_s[i - 2], p.d, lane, f);
                }
            }
        if (fresh < 0 && tid == 0 && g == 0) atomicOr(p.status, TBL_DEV_CACHE_FULL);
        __syncthreads();
    }
    // queries: B fragments of every step, two rows (2 t4, 2 t4 + 1) of factors
    uint32_t q[NT][kBlocks][4][2];
    float c[NT][2];
    int last[NT][2];                                             // last token each row of the scores' fragments sees
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const int at = first + 8 * u + g8, ok = at < total, r = ok ? at : 0;
        const __half* src = kWhole ? q_s[kWhole ? 8 * u + g8 : 0]
                                   : static_cast<const __half*>(p.q) + ((static_cast<size_t>(seq) * p.n_tok + r / p.group) * p.H + g * p.group + r % p.group) * DP;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint2 v = *reinterpret_cast<const uint2*>(src + 64 * b + 16 * t4 + 4 * s);
                q[u][b][s][0] = ok ? v.x : 0u;
                q[u][b][s][1] = ok ? v.y : 0u;
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = min(first + 8 * u + 2 * t4 + e, total - 1);
            c[u][e] = p.scale_log2 * (kWhole ? factor_s[row] : p.q_factor[(static_cast<size_t>(seq) * p.n_tok + row / p.group) * p.H + g * p.group + row % p.group]);
            last[u][e] = min(pos0 + row / p.group, t1 - 1);
        }
    }
    const int all_see = min(pos0 + first / p.group, t1 - 1);     // the last token that every row sees
    float o[kBlocks * 4][NT][4];
#pragma unroll
    for (int i = 0; i < kBlocks * 4; ++i)
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][u][e] = 0.0f;
    float mx[NT][2], sum[NT][2];
#pragma unroll
    for (int u = 0; u < NT; ++u) { mx[u][0] = mx[u][1] = -FLT_MAX; sum[u][0] = sum[u][1] = 0.0f; }
    const uint32_t key_byte = t4 | (4 + t4) << 4, value_byte = (g8 >> 1) | (4 + (g8 >> 1)) << 4;   // that byte of either word
    const int ka = token_of(g8), va = token_of(2 * t4), vb = token_of(2 * t4 + 1);               // MMA rows 8 .. 15: one token further on
    bool alive = true;
    uint32_t phase = 0;
    int stage = 0;
    for (int t = begin; t < t1; t += step) {
        // (after a wait that gave up nothing more is asked for, and what is on its way gets a short time)
        alive = __all_sync(0xffffffffu, mbar_wait_bounded(&full[warp][stage], phase, p.status, alive ? kWaitSpinLimit : 1024)) && alive;
        const uint32_t tile = smem_u32(ring + stage * L::kTileBytes);
        if (kWhole && fresh >= t && fresh < t + kTile) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(ring + stage * L::kTileBytes + (fresh - t) * L::kRow);
            for (int i = lane; i < L::kRow / 4; i += 32) dst[i] = reinterpret_cast<const uint32_t*>(fresh_s)[i];
            __syncwarp();
        }
        float s[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[h][u][e] = 0.0f;
            const uint32_t row = tile + (16 * h + ka) * L::kRow;
            uint32_t sx4[kBlocks], sy4[kBlocks];                 // scales of a block, a byte each
            lds_words<kBlocks>(row + DP, sx4);
            lds_words<kBlocks>(row + L::kRow + DP, sy4);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const uint2 x = lds64(row + 32 * b + 8 * t4), y = lds64(row + L::kRow + 32 * b + 8 * t4);
                const __half2 both = scales_of(__byte_perm(sx4[b], sy4[b], key_byte));
                const __half2 sx = __low2half2(both), sy = __high2half2(both);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint32_t a[4], k[4];
                    widen(w ? x.y : x.x, sx, a);
                    widen(w ? y.y : y.x, sy, k);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int u = 0; u < NT; ++u)
                            mma_f16(s[h][u], a[2 * e], k[2 * e], a[2 * e + 1], k[2 * e + 1], q[u][b][2 * w + e][0], q[u][b][2 * w + e][1]);
                }
            }
        }
        const bool whole = t + kTile - 1 <= all_see;             // nothing of the tile is masked
        float top[NT][2];
        bool grown = false;
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x[4];                                      // tokens ka, ka + 1 of either half
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = s[i >> 1][u][2 * (i & 1) + e] * c[u][e];
                    if (!whole && t + 16 * (i >> 1) + ka + (i & 1) > last[u][e]) x[i] = -INFINITY;
                    s[i >> 1][u][2 * (i & 1) + e] = x[i];
                }
                top[u][e] = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                grown = grown || top[u][e] > mx[u][e] + kRescale;
            }
        // the maximum only moves when it grows by 2^4, so that lanes need not ask each other for most tiles; then output and sum are rescaled
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = top[u][e];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    m = m > mx[u][e] + kRescale ? m : mx[u][e];
                    f[e] = ex2(mx[u][e] - m);
                    mx[u][e] = m;
                    sum[u][e] *= f[e];
                }
#pragma unroll
                for (int i = 0; i < kBlocks * 4; ++i) { o[i][u][0] *= f[0]; o[i][u][1] *= f[1]; o[i][u][2] *= f[0]; o[i][u][3] *= f[1]; }
            }
        }
        uint32_t pt[2][NT][2];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i >> 1][u][2 * (i & 1) + e] = x[i] = ex2(s[i >> 1][u][2 * (i & 1) + e] - (mx[u][e] - kTop));
                sum[u][e] += (x[0] + x[1]) + (x[2] + x[3]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const __half2 w = __floats2half2_rn(s[h][u][2 * r], s[h][u][2 * r + 1]);
                    pt[h][u][r] = transposed(*reinterpret_cast<const uint32_t*>(&w));
                }
        }
        // rows nobody has written may hold anything: a weight of zero needs a finite value beside it (the split's last tile: nothing is loaded over
        // it any more)
        if (t + kTile > t1) {
            if (t + lane >= t1)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<uint32_t*>(ring + stage * L::kTileBytes + lane * L::kRow + DP + DP / 16 + 4 * b) = 0;
            __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // MMA columns 2 t4, 2 t4 + 1 are tokens va, vb, columns 2 t4 + 8, 2 t4 + 9 the ones behind them
            const uint32_t ra = tile + (16 * h + va) * L::kRow, rb = tile + (16 * h + vb) * L::kRow;
            const uint32_t codes = DP / 2 + 4 * g8, scale = DP + DP / 16;
            uint32_t sa4[2][kBlocks], sb4[2][kBlocks];
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                lds_words<kBlocks>(ra + d * L::kRow + scale, sa4[d]);
                lds_words<kBlocks>(rb + d * L::kRow + scale, sb4[d]);
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                uint32_t a[2][8];
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    const uint32_t wa = lds32(ra + d * L::kRow + codes + 32 * b), wb = lds32(rb + d * L::kRow + codes + 32 * b);
                    const __half2 sc = scales_of(__byte_perm(sa4[d][b], sb4[d][b], value_byte));
                    uint32_t even[4], odd[4];
                    widen((wa & 0x0f0f0f0fu) | ((wb << 4) & 0xf0f0f0f0u), sc, even);
                    widen(((wa >> 4) & 0x0f0f0f0fu) | (wb & 0xf0f0f0f0u), sc, odd);
#pragma unroll
                    for (int i = 0; i < 4; ++i) { a[d][2 * i] = even[i]; a[d][2 * i + 1] = odd[i]; }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < NT; ++u) mma_f16(o[4 * b + i][u], a[0][2 * i], a[0][2 * i + 1], a[1][2 * i], a[1][2 * i + 1], pt[h][u][0], pt[h][u][1]);
            }
        }
        __syncwarp();                                            // the tile is no longer read
        if (alive) load_tile(stage, t + kStages * step);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
    __syncthreads();                                             // tiles are done with: their room takes the outputs
    pdl_launch_dependents();
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = sum[u][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            if (g8 == 0) { m_s[warp][8 * u + 2 * t4 + e] = mx[u][e]; l_s[warp][8 * u + 2 * t4 + e] = l; }
            float* dst = o_s + (warp * kRows + 8 * u + 2 * t4 + e) * L::kLdo + 8 * g8;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    *reinterpret_cast<float4*>(dst + 64 * b + 2 * i) =
                        make_float4(o[4 * b + i][u][e], o[4 * b + i][u][2 + e], o[4 * b + i + 1][u][e], o[4 * b + i + 1][u][2 + e]);
        }
    __syncthreads();
    // the warps come together: sums of this split, over the first warp's
    const int rows = min(kRows, total - first);
    for (int i = tid; i < rows * (DP / 4); i += kThreads) {
        const int r = i / (DP / 4), col = (i % (DP / 4)) * 4;
        float top = m_s[0][r];
#pragma unroll
        for (int k = 1; k < W; ++k) top = fmaxf(top, m_s[k][r]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float w = ex2(m_s[k][r] - top);
            const float4 x = *reinterpret_cast<const float4*>(o_s + (k * kRows + r) * L::kLdo + col);
            v.x = fmaf(x.x, w, v.x); v.y = fmaf(x.y, w, v.y); v.z = fmaf(x.z, w, v.z); v.w = fmaf(x.w, w, v.w);
            l = fmaf(l_s[k][r], w, l);
        }
        *reinterpret_cast<float4*>(o_s + r * L::kLdo + col) = v;
        if (col == 0) { top_s[r] = top; sum_s[r] = l; }
    }
    __syncthreads();
    if (p.splits > 1) {
        for (int i = tid; i < rows * p.d; i += kThreads) {
            const int r = i / p.d, col = i - r * p.d, row = first + r;
            const size_t u = ((static_cast<size_t>(seq) * p.n_tok + row / p.group) * p.H + g * p.group + row % p.group) * p.splits + split;
            if (col == 0) { p.part_m[u] = top_s[r]; p.part_l[u] = sum_s[r]; }
            p.part_o[u * p.ldo + col] = o_s[r * L::kLdo + col];
        }
        return;
    }
    for (int i = tid; i < rows * p.d; i += kThreads) {
        const int r = i / p.d, col = i - r * p.d, at = first + r, head = g * p.group + at % p.group;
        const size_t row = static_cast<size_t>(seq) * p.n_tok + at / p.group;
        const float gate = p.g_off < 0 ? 1.0f : sigmoid_f(p.proj[row * p.ld + p.g_off + head * p.d + col]);
        static_cast<bf16*>(p.out)[(row * p.H + head) * p.d + col] = __float2bfloat16_rn(o_s[r * L::kLdo + col] * (p.value_unit / sum_s[r]) * gate);
    }
}

// blocks of query rows: 16 at a time halves the trips over the cache, but a head of more than 128 has no registers for it
int rows_of(int dim, int total) { return total > 8 && dim <= 128 ? 16 : 8; }

template <int DP, int NT, int W, int V>
cudaError_t launch(const QuantizedParams& p, int n_seq, cudaStream_t st) {
    static bool done[64] = {};
    const dim3 grid(n_seq * p.G, ceil_div(static_cast<long long>(p.n_tok) * p.group, 8 * NT), p.splits);
    if (grid.y > 65535 || grid.z > 65535) return cudaErrorInvalidValue;
    constexpr size_t smem = Layout<DP, NT, W>::kBytes;
    const cudaError_t e = allow_smem(quantized_stream_kernel<DP, NT, W, V>, smem, done);
    if (e != cudaSuccess) return e;
    return launch_dependent(quantized_stream_kernel<DP, NT, W, V>, grid, dim3(32 * W), smem, st, p);
}
template <int DP, int NT>
cudaError_t launch_plan(const QuantizedParams& p, const StreamPlan& plan, int vec, int n_seq, cudaStream_t st) {
    if constexpr (DP <= 128) {
        if (plan.warps == 16) return !plan.whole ? launch<DP, NT, 16, 0>(p, n_seq, st) : vec ? launch<DP, NT, 16, 4>(p, n_seq, st) : launch<DP, NT, 16, 1>(p, n_seq, st);
    }
    return !plan.whole ? launch<DP, NT, 4, 0>(p, n_seq, st) : vec ? launch<DP, NT, 4, 4>(p, n_seq, st) : launch<DP, NT, 4, 1>(p, n_seq, st);
}

}  // namespace

int quantized_stream_rows(const tbl_quantized_mixer& m, int n_tok) {
    const long long total = static_cast<long long>(n_tok) * (m.heads / m.kv_heads);
    return rows_of(m.dim, static_cast<int>(total < 64 ? total : 64));
}

StreamPlan quantized_stream_plan(const tbl_quantized_mixer& m, int n_seq, int n_tok, int context) {
    const long long total = static_cast<long long>(n_tok) * (m.heads / m.kv_heads);
    const int rows = quantized_stream_rows(m, n_tok);
    const long long units = static_cast<long long>(n_seq) * m.kv_heads * ceil_div(total, rows);
    StreamPlan w{4, 1, 1, 0};
    const int tokens = ceil_div(context, 4 * kTile);             // a split is worth at least a tile of each warp
    long long s = 4LL * kNumSm / units;                          // four CTAs of four warps to an SM
    if (s > tokens) s = tokens;
    if (s > 1024) s = 1024;
    w.splits = w.most = s < 1 ? 1 : static_cast<int>(s);
    // Instead of splits, whose sums another kernel joins: one CTA of sixteen warps an SM.  In the time of a tile (1.7 us with sixteen warps to an
    // SM): what a warp takes one after the other, and 1.4 tiles for the other kernel, more with its blocks (a 64th for a unit up to 80) and splits (a
    // 20th each).  One token of 32 and 8 heads, sixteen warps and splits: one sequence over 900 9.7 and 9.8 us, 2000 13.2 and 10.6, 8192 33.5 and
    // 14.7; 8 over 2048 13.9 and 15.0, 4096 20.7 and 18.7; 18 over 4096 22 and 27; 30 over 4096 43 and 45.
    if (w.splits > 1 && m.dim <= 128) {
        const double wide = ceil_div(context, 16 * kTile) * static_cast<double>(ceil_div(units, kNumSm));
        const double split = ceil_div(context, 4LL * kTile * w.splits) + 1.4 + (units < 80 ? units : 80) / 64.0 + w.splits / 20.0;
        if (wide <= split) { w.warps = 16; w.splits = 1; }
    }
    // As a whole one launch less, but fewer CTAs to an SM, whose own chains before the first tile show once they take turns (64 sequences of 8 heads
    // over 4096 tokens 82 and 72 us, over 600 26 and 20, 37 over 4096 46 and 44)
    w.whole = n_tok == 1 && w.splits == 1 && total <= rows && units <= (w.warps == 16 ? 1 : 2) * kNumSm;
    return w;
}

int launch_quantized_stream(const QuantizedParams& p, const StreamPlan& plan, int vec, int n_seq, cudaStream_t st) {
    const long long total = static_cast<long long>(p.n_tok) * p.group;
    const bool two = rows_of(p.d, static_cast<int>(total < 64 ? total : 64)) == 16;
    cudaError_t e;
    switch (p.width) {
        case 64: e = two ? launch_plan<64, 2>(p, plan, vec, n_seq, st) : launch_plan<64, 1>(p, plan, vec, n_seq, st); break;
        case 128: e = two ? launch_plan<128, 2>(p, plan, vec, n_seq, st) : launch_plan<128, 1>(p, plan, vec, n_seq, st); break;
        case 192: e = launch_plan<192, 1>(p, plan, vec, n_seq, st); break;
        default: e = launch_plan<256, 1>(p, plan, vec, n_seq, st); break;
    }
    return e == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

}  // namespace stack
}  // namespace tbl
