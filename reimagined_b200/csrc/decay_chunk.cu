// Linear attention with decay over prompts, by chunks of 128 tokens on the tensor cores (tcgen05).
//
// With y = exp(log_decay) and S the state before a chunk, the token i of the chunk (from 0 on) has
//   o_i = scale (sum_{j <= i} y^(i-j) (q_i . k_j) v_j + y^(i+1) S q_i),      S' = y^n S + sum_j y^(n-1-j) v_j k_j^T.
//
//   decay_sums_kernel    the last sum of every chunk: no chunk waits for another
//   decay_join_kernel    the states before the chunks one after the other, element by element in fp32
//   decay_chunk_kernel   the outputs of every chunk: two products for the tokens inside, one for the state
// Queries and keys are normed and turned where they are read, from the fp32 projections: what has to pass through memory is the projections, twice for keys and
// values.  A long prompt goes by pieces whose projections and sums stay in the second-level cache between the three kernels.
//
// Precision.  The states are sums over the whole sequence and stay fp32: their products take both operands as three bf16 terms each (24 bits; six products, the
// five small ones in an accumulator of their own, so that what the tensor core's sums cut off is of their size).  Outputs are rounded to bf16, so their operands are
// fp16 under a power of two for every token, and for every row of a state (errors of 2^-12; keys, values and weights y^(i-j) share the smallest of their
// factors of a chunk, which only costs numbers 2^-14 below the chunk's largest their last bits).
#include <cuda_fp16.h>

#include "decay.cuh"
#include "flash.cuh"

namespace tbl {
namespace stack {
namespace {

using namespace tc05;

constexpr int kTokens = 128, kThreads = 256, kWarps = kThreads / 32;
constexpr int kSub = 128 * 128;                  // 128 rows of 64 sixteen-bit numbers, 128-byte swizzle
constexpr int kBox = 64 * 128;                   // 64 tokens of the same
constexpr uint32_t kTransposeA = 1u << 15, kTransposeB = 1u << 16;

struct ChunkParams {
    DecayParams d;
    float* sums;                 // [unit][chunk of the piece][key / 4][value][4]
    uint8_t* images;             // [unit][chunk]: the state before it as the B operand [value][key] of fp16, as it lies in shared memory
    float* scales;               // [unit][chunk][value]: the power of two its rows were divided by
    const float* states;         // before the piece
    int first, chunks;           // first token of the piece, its chunks for each sequence
};

// sixteen-bit operands that lie with neighbours of the M or N side together: rows of 64 (128 bytes, swizzled), a row per token, groups of 8 tokens 1024 bytes
// apart, the next 64 columns `box` bytes further on
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr, int box) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(box / 16) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// place of column c of row r in tiles of 64 columns, `tile` bytes each
__device__ __forceinline__ uint32_t swizzled(int r, int c, int tile) { return (c >> 6) * tile + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4) + (c & 7) * 2; }

template <int V>
__device__ __forceinline__ void put_halves(uint8_t* base, int r, int c, int tile, const float* v, float f) {
    uint8_t* dst = base + swizzled(r, c, tile);
    if (V == 4) {
        const __half2 a = __floats2half2_rn(v[0] * f, v[V > 1 ? 1 : 0] * f), b = __floats2half2_rn(v[V > 2 ? 2 : 0] * f, v[V > 3 ? 3 : 0] * f);
        *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        *reinterpret_cast<__half*>(dst) = __float2half_rn(v[0] * f);
    }
}
// three bf16 terms of each number, in three tiles `piece` bytes apart
template <int V>
__device__ __forceinline__ void put_terms(uint8_t* base, int r, int c, int tile, int piece, const float* v, float f) {
    uint8_t* dst = base + swizzled(r, c, tile);
    float x[4];
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = v[e] * f;
#pragma unroll
    for (int t = 0; t < 3; ++t) {
        if (V == 4) {
            const uint32_t a = pack_bf16(x[0], x[V > 1 ? 1 : 0]), b = pack_bf16(x[V > 2 ? 2 : 0], x[V > 3 ? 3 : 0]);
            *reinterpret_cast<uint2*>(dst + t * piece) = make_uint2(a, b);
            x[0] -= bf_lo(a); x[V > 1 ? 1 : 0] -= bf_hi(a); x[V > 2 ? 2 : 0] -= bf_lo(b); x[V > 3 ? 3 : 0] -= bf_hi(b);
        } else {
            const bf16 a = __float2bfloat16_rn(x[0]);
            *reinterpret_cast<bf16*>(dst + t * piece) = a;
            x[0] -= __bfloat162float(a);
        }
    }
}

// How a token's head lies over the lanes of a warp: LPH lanes for a token, 32 / LPH tokens side by side.
template <int DP, int V>
struct Lanes {
    static constexpr int kLph = V == 4 ? DP / 8 : 32, kSide = 32 / kLph;
    using Units = HeadUnits<V, kLph>;
};

__device__ __forceinline__ Rotation unturned() { return Rotation{nullptr, nullptr, 0, 0, 0}; }

// largest number of a head over its lanes, as a power of two (1 for a head of zeros)
template <int LPH, typename U>
__device__ __forceinline__ float power_of(const U& x) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < U::kUnits; ++i)
#pragma unroll
        for (int e = 0; e < static_cast<int>(sizeof(x.x[0]) / 4); ++e) most = fmaxf(most, fabsf(x.x[i][e]));
#pragma unroll
    for (int o = LPH / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const uint32_t power = min(__float_as_uint(most) >> 23, 253u);
    return power ? __uint_as_float(power << 23) : 1.0f;
}
__device__ __forceinline__ float inverse_power(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }

struct Place {
    int unit, seq, head, chunk, first, n, slot, pos0;    // first: token of the sequence's portion; n: tokens of the chunk
};
__device__ __forceinline__ Place place_of(const ChunkParams& c, int unit, int chunk) {
    Place a;
    a.unit = unit; a.seq = unit / c.d.H; a.head = unit % c.d.H; a.chunk = chunk;
    a.first = c.first + chunk * kTokens;
    a.n = min(kTokens, c.d.n_tok - a.first);
    a.slot = c.d.slots[a.seq];
    a.pos0 = c.d.positions[a.slot] + a.first;
    return a;
}
__device__ __forceinline__ int table_row(const DecayParams& p, int pos) { return p.r.half > 0 ? min(max(pos, 0), p.r.positions - 1) : 0; }

// ---- sums of the chunks -----------------------------------------------------------------------------------------------------------------
// One CTA per (unit, chunk): D[value][key] = sum over tokens, M = 128 values (of which DP count), N = DP keys, two tiles of 64 tokens; both operands lie as they come, a row
// per token.  Bound by memory and by the cutting of numbers into terms; two CTAs to an SM.
template <int DP, int V>
__global__ void __launch_bounds__(kThreads, 2) decay_sums_kernel(const ChunkParams c) {
    using Ln = Lanes<DP, V>;
    constexpr int kPiece = DP / 64 * kBox, kPerWarp = 64 / kWarps, kRounds = kPerWarp / Ln::kSide;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t done;
    __shared__ uint32_t tmem_slot;
    uint8_t *k_s = smem, *v_s = smem + 3 * kPiece;       // three terms each (the values' last tile may be read past its end: room for that is behind)
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const DecayParams& p = c.d;
    if (threadIdx.x == 0) {
        mbar_init(&done, 1);
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (p.d != DP)                                       // columns nobody writes
        for (int i = threadIdx.x; i < 6 * kPiece / 16; i += kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();                             // (after the allocation: a dependent's would otherwise stand in its way)
    pdl_wait();
    const Place a = place_of(c, blockIdx.y, blockIdx.x);
    const float rate = p.log_decay[a.head];
    const int group = lane / Ln::kLph, gl = lane % Ln::kLph;
    const float* base = p.proj + (static_cast<size_t>(a.seq) * p.n_tok + a.first) * p.ld + a.head * p.d;
    if (p.r.half > 0 && threadIdx.x == 0 && (a.pos0 < 0 || a.pos0 + a.n > p.r.positions)) atomicOr(p.status, TBL_DEV_CACHE_FULL);
    bool alive = true;
    const int tiles = (a.n + 63) / 64;
    for (int tile = 0; tile < tiles; ++tile) {
        typename Ln::Units k[kRounds], v[kRounds];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int j = tile * 64 + warp * kPerWarp + i * Ln::kSide + group, n = j < a.n ? p.d : 0;
            const float* src = base + static_cast<size_t>(min(j, a.n - 1)) * p.ld;
            k[i].load(p.r, src + p.H * p.d, n, gl);
            v[i].load(unturned(), src + p.v_off, n, gl);
        }
        if (tile) alive = mbar_wait_bounded(&done, 0, p.status);          // the first tile's products have read their operands
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int r = warp * kPerWarp + i * Ln::kSide + group, j = tile * 64 + r;
            k[i].template turn<float>(p.r, p.k_norm, p.eps, table_row(p, a.pos0 + min(j, a.n - 1)), p.d, gl);
            if (j >= a.n) {                              // (the norm of nothing may be 0 / 0)
#pragma unroll
                for (int u = 0; u < Ln::Units::kUnits; ++u)
#pragma unroll
                    for (int e = 0; e < 2 * V; ++e) k[i].x[u][e] = 0.0f;
            }
            const float f = j < a.n - 1 ? expf(rate * static_cast<float>(a.n - 1 - j)) : 1.0f;
#pragma unroll
            for (int u = 0; u < Ln::Units::kUnits; ++u) {
                int x, y;
                Ln::Units::runs(p.r, gl + Ln::kLph * u, x, y);
                if (x < p.d) put_terms<V>(k_s, r, x, kBox, kPiece, k[i].x[u], 1.0f);
                if (y < p.d) put_terms<V>(k_s, r, y, kBox, kPiece, k[i].x[u] + V, 1.0f);
                Ln::Units::runs(unturned(), gl + Ln::kLph * u, x, y);
                if (x < p.d) put_terms<V>(v_s, r, x, kBox, kPiece, v[i].x[u], f);
                if (y < p.d) put_terms<V>(v_s, r, y, kBox, kPiece, v[i].x[u] + V, f);
            }
        }
        fence_proxy_async();
        __syncthreads();
        if (warp == 0 && elect_one() && alive) {
            tc_fence_after();
            const uint32_t id = idesc_bf16(DP) | kTransposeA | kTransposeB;
            const uint64_t vd = desc_rows(smem_u32(v_s), kBox), kd = desc_rows(smem_u32(k_s), kBox);
            constexpr int kStep = kPiece / 16;
#pragma unroll
            for (int s = 0; s < 4; ++s) {                // 16 tokens each; terms whose orders add up to 2 and 1 first
                const uint32_t more = tile | s;
                umma_f16(tmem + DP, vd + 2 * kStep + 128 * s, kd + 128 * s, id, more);
                umma_f16(tmem + DP, vd + 128 * s, kd + 2 * kStep + 128 * s, id, 1);
                umma_f16(tmem + DP, vd + kStep + 128 * s, kd + kStep + 128 * s, id, 1);
                umma_f16(tmem + DP, vd + kStep + 128 * s, kd + 128 * s, id, 1);
                umma_f16(tmem + DP, vd + 128 * s, kd + kStep + 128 * s, id, 1);
                umma_f16(tmem, vd + 128 * s, kd + 128 * s, id, more);
            }
            umma_commit(&done);
        }
    }
    alive = mbar_wait_bounded(&done, (tiles - 1) & 1, p.status) && alive;
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;              // value
    if (alive && (warp & 3) * 32 < DP) {
        float* dst = c.sums + (static_cast<size_t>(a.unit) * c.chunks + a.chunk) * DP * DP;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
#pragma unroll
        for (int q = 0; q < DP / 64; ++q) {
            const int col = (warp >> 2) * (DP / 2) + 32 * q;
            uint32_t x[32], y[32];
            tmem_ld32(tmem + lanes + col, x);
            tmem_ld32(tmem + lanes + DP + col, y);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                float4 f;
                f.x = __uint_as_float(x[e]) + __uint_as_float(y[e]);
                f.y = __uint_as_float(x[e + 1]) + __uint_as_float(y[e + 1]);
                f.z = __uint_as_float(x[e + 2]) + __uint_as_float(y[e + 2]);
                f.w = __uint_as_float(x[e + 3]) + __uint_as_float(y[e + 3]);
                reinterpret_cast<float4*>(dst)[(col + e) / 4 * DP + row] = f;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
    }
}

// ---- states before the chunks -----------------------------------------------------------------------------------------------------------
// DP / 8 lanes share a row (a value's keys), eight neighbouring keys each.
template <int DP>
__global__ void __launch_bounds__(128) decay_join_kernel(const ChunkParams c) {
    constexpr int kLph = DP / 8, kSide = 32 / kLph;
    pdl_launch_dependents();
    pdl_wait();
    const DecayParams& p = c.d;
    const int lane = threadIdx.x & 31, gl = lane % kLph, row = (blockIdx.x * 4 + (threadIdx.x >> 5)) * kSide + lane / kLph, unit = blockIdx.y;
    const int seq = unit / p.H, head = unit % p.H;
    const size_t state = (static_cast<size_t>(p.slots[seq]) * p.H + head) * p.d * p.d + static_cast<size_t>(row) * p.d;
    const float rate = p.log_decay[head];
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = row < p.d && 8 * gl + e < p.d ? c.states[state + 8 * gl + e] : 0.0f;
    const float4* src = reinterpret_cast<const float4*>(c.sums + static_cast<size_t>(unit) * c.chunks * DP * DP) + 2 * gl * DP + row;
    constexpr int kAhead = 4;
    float4 x[kAhead][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < c.chunks) { x[i][0] = src[static_cast<size_t>(i) * DP * DP / 4]; x[i][1] = src[static_cast<size_t>(i) * DP * DP / 4 + DP]; }
    const float less = expm1f(rate * static_cast<float>(kTokens));
    for (int i0 = 0; i0 < c.chunks; i0 += kAhead) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k;
            if (i >= c.chunks) break;
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(s[e]));
#pragma unroll
            for (int o = kLph / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const uint32_t bits = min(__float_as_uint(most) >> 23, 253u);
            const float power = bits ? __uint_as_float(bits << 23) : 1.0f, inv = inverse_power(power);
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __half2 w = __floats2half2_rn(s[2 * e] * inv, s[2 * e + 1] * inv);
                h[e] = *reinterpret_cast<const uint32_t*>(&w);
            }
            const size_t at = static_cast<size_t>(unit) * c.chunks + i;
            *reinterpret_cast<uint4*>(c.images + at * DP * DP * 2 + swizzled(row, 8 * gl, DP * 128)) = make_uint4(h[0], h[1], h[2], h[3]);
            if (gl == 0) c.scales[at * DP + row] = power;
            const int n = min(kTokens, p.n_tok - c.first - i * kTokens);
            const float l = n == kTokens ? less : expm1f(rate * static_cast<float>(n));
            const float4 u = x[k][0], v = x[k][1];
            s[0] = fmaf(l, s[0], s[0]) + u.x; s[1] = fmaf(l, s[1], s[1]) + u.y; s[2] = fmaf(l, s[2], s[2]) + u.z; s[3] = fmaf(l, s[3], s[3]) + u.w;
            s[4] = fmaf(l, s[4], s[4]) + v.x; s[5] = fmaf(l, s[5], s[5]) + v.y; s[6] = fmaf(l, s[6], s[6]) + v.z; s[7] = fmaf(l, s[7], s[7]) + v.w;
            if (i + kAhead < c.chunks) {
                x[k][0] = src[static_cast<size_t>(i + kAhead) * DP * DP / 4];
                x[k][1] = src[static_cast<size_t>(i + kAhead) * DP * DP / 4 + DP];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (row < p.d && 8 * gl + e < p.d) p.next[state + 8 * gl + e] = s[e];
}

// ---- outputs of the chunks ----------------------------------------------------------------------------------------------------------------
// One CTA per (unit, chunk).  Scores Q K^T in the first 128 columns of its tensor memory, weights in their place (fp16, the A operand of the second product), the
// tokens' part of the outputs behind them, then the state's part over the weights.  The state's operand comes by one bulk copy into the keys' room.  Outputs are
// collected in shared memory, so that gates are read and rows are written whole.
template <int DP, int V>
__global__ void __launch_bounds__(kThreads, 2) decay_chunk_kernel(const ChunkParams c) {
    using Ln = Lanes<DP, V>;
    constexpr int kTile = DP / 64 * kSub, kPerWarp = kTokens / kWarps, kLdo = DP + 4, kImage = DP * DP * 2;
    // rounds of loads in flight at once
    constexpr int kRounds = kPerWarp / Ln::kSide, kFlight = V == 4 ? (kRounds < 4 ? kRounds : 4) : 2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ float power_s[kTokens + 1];               // y^n
    __shared__ float q_f[kTokens], kv_f[kTokens], v_f[kTokens], scale_s[DP], ss_s[2][kTokens], most_s;
    __shared__ __align__(8) uint64_t bars[3];            // scores, state's image, outputs
    __shared__ uint32_t tmem_slot;
    uint8_t *q_s = smem, *k_s = smem + kTile, *v_s = smem + 2 * kTile;
    float* o_s = reinterpret_cast<float*>(smem);         // afterwards: [token][kLdo]
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const DecayParams& p = c.d;
    if (tid == 0) {
        for (int i = 0; i < 3; ++i) mbar_init(&bars[i], 1);
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (p.d != DP)
        for (int i = tid; i < 3 * kTile / 16; i += kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();
    const Place a = place_of(c, blockIdx.y, blockIdx.x);
    const size_t at = static_cast<size_t>(a.unit) * c.chunks + a.chunk;
    const float rate = p.log_decay[a.head];
    if (tid <= kTokens) power_s[tid] = tid ? expf(rate * static_cast<float>(tid)) : 1.0f;
    if (tid < DP) scale_s[tid] = c.scales[at * DP + tid];
    const int group = lane / Ln::kLph, gl = lane % Ln::kLph;
    const float* base = p.proj + (static_cast<size_t>(a.seq) * p.n_tok + a.first) * p.ld + a.head * p.d;
#pragma unroll 1
    for (int what = 0; what < 3; ++what) {               // queries, keys, values
        const Rotation r = what < 2 ? p.r : unturned();
        const float* src = base + (what == 0 ? 0 : what == 1 ? p.H * p.d : p.v_off);
        const float* norm = what == 0 ? p.q_norm : p.k_norm;
        uint8_t* dst = smem + what * kTile;
#pragma unroll 1
        for (int i0 = 0; i0 < kRounds; i0 += kFlight) {
            typename Ln::Units x[kFlight];
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const int j = warp * kPerWarp + (i0 + i) * Ln::kSide + group;
                x[i].load(r, src + static_cast<size_t>(min(j, a.n - 1)) * p.ld, j < a.n ? p.d : 0, gl);
            }
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const int j = warp * kPerWarp + (i0 + i) * Ln::kSide + group;
                if (what < 2) x[i].template turn<float>(r, norm, p.eps, table_row(p, a.pos0 + min(j, a.n - 1)), p.d, gl);
                const float power = power_of<Ln::kLph>(x[i]), inv = inverse_power(power);
                if (gl == 0) (what == 0 ? q_f : what == 1 ? kv_f : v_f)[j] = power;
#pragma unroll
                for (int u = 0; u < Ln::Units::kUnits; ++u) {
                    int y, z;
                    Ln::Units::runs(r, gl + Ln::kLph * u, y, z);
                    if (y < p.d) put_halves<V>(dst, j, y, kSub, x[i].x[u], inv);
                    if (z < p.d) put_halves<V>(dst, j, z, kSub, x[i].x[u] + V, inv);
                }
            }
        }
    }
    fence_proxy_async();
    __syncthreads();
    bool alive = true;
    if (warp == 0) {
        if (elect_one()) {
            tc_fence_after();
            flash::products(tmem, smem_desc_sw128(smem_u32(q_s)), smem_desc_sw128(smem_u32(k_s)), DP / 16, idesc_f16(kTokens), 0);
            umma_commit(&bars[0]);
        }
        __syncwarp();
    } else if (warp == 1) {                              // the largest factor of a token's key and value together
        float f[kTokens / 32], most = 0.0f;
#pragma unroll
        for (int i = 0; i < kTokens / 32; ++i) {
            const int j = lane + 32 * i;
            // (as exponents: the product of two powers of two may pass the ends of fp32)
            f[i] = static_cast<float>(static_cast<int>(__float_as_uint(kv_f[j]) >> 23) + static_cast<int>(__float_as_uint(v_f[j]) >> 23));
            if (j >= a.n) f[i] = 0.0f;
            most = fmaxf(most, f[i]);
        }
        most = warp_max(most);
#pragma unroll
        for (int i = 0; i < kTokens / 32; ++i) kv_f[lane + 32 * i] = exp2f(f[i] - most);
        if (lane == 0) most_s = most - 254.0f;
    }
    __syncthreads();
    alive = mbar_wait_bounded(&bars[0], 0, p.status);
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    if (alive && warp == 0 && elect_one()) {             // the keys are done with
        mbar_arrive_expect_tx(&bars[1], kImage);
        bulk_g2s(k_s, c.images + at * kImage, kImage, &bars[1]);
    }
    __syncwarp();
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
#pragma unroll 1
    for (int ch = 2 * half; ch < 2 * half + 2; ++ch) {
        uint32_t x[32], y[16];
        if (ch * 32 > (warp & 3) * 32 + 31) {            // nothing of it is visible to these rows
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = 0;
        } else {
            tmem_ld32(tmem + lanes + ch * 32, x);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int j = ch * 32 + 2 * e + k;
                    w[k] = j <= row ? __uint_as_float(x[2 * e + k]) * power_s[max(row - j, 0)] * kv_f[j] : 0.0f;
                }
                const __half2 h = __floats2half2_rn(w[0], w[1]);
                y[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        tmem_st16(tmem + lanes + ch * 32, y);
    }
    tmem_st_wait();
    tc_fence_before();
    __syncthreads();
    if (alive && warp == 0 && elect_one()) {
        tc_fence_after();
        const uint64_t vd = desc_rows(smem_u32(v_s), kSub);
        const uint32_t id = idesc_f16(DP) | kTransposeB;
#pragma unroll
        for (int k = 0; k < kTokens / 16; ++k) umma_f16_ta(tmem + kTokens, tmem + (k >> 1) * 32 + (k & 1) * 8, vd + 128 * k, id, k != 0);
        const bool image = mbar_wait_bounded(&bars[1], 0, p.status);
        if (image) flash::products(tmem, smem_desc_sw128(smem_u32(q_s)), smem_desc_sw128(smem_u32(k_s)), DP / 16, idesc_f16(DP), 0);
        umma_commit(&bars[2]);
    }
    __syncwarp();
    if (alive) alive = mbar_wait_bounded(&bars[2], 0, p.status);
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    // a row's halves are two threads'; the sums of squares meet in shared memory
    const float f = q_f[row] * p.scale, inside = f * exp2f(most_s), before = f * power_s[min(row + 1, kTokens)];
    float ss = 0.0f;
#pragma unroll 1
    for (int q = 0; q < DP / 64; ++q) {
        const int col = half * (DP / 2) + 32 * q;
        uint32_t x[32], y[32];
        tmem_ld32(tmem + lanes + kTokens + col, x);
        tmem_ld32(tmem + lanes + col, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            float o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[k] = fmaf(__uint_as_float(x[e + k]), inside, __uint_as_float(y[e + k]) * (before * scale_s[col + e + k]));
                if (col + e + k < p.d) ss = fmaf(o[k], o[k], ss);
            }
            *reinterpret_cast<float4*>(o_s + row * kLdo + col + e) = make_float4(o[0], o[1], o[2], o[3]);
        }
    }
    ss_s[half][row] = ss;
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
    }
    if (!alive) return;
    bf16* out = static_cast<bf16*>(p.out) + ((static_cast<size_t>(a.seq) * p.n_tok + a.first) * p.H + a.head) * p.d;
    const float* gate = p.g_off < 0 ? nullptr : base + p.g_off;
    const float* norm = p.norm ? p.norm + a.head * p.d : nullptr;
    const bool vec = p.vec && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 && (reinterpret_cast<uintptr_t>(p.norm) & 15) == 0;
    if (vec) {
        constexpr int kLanes = DP / 4;                   // lanes to a row
        const int col = (tid % kLanes) * 4;
        float4 w = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (norm && col < p.d) w = *reinterpret_cast<const float4*>(norm + col);
        if (col < p.d) {
#pragma unroll 4
            for (int j = tid / kLanes; j < a.n; j += kThreads / kLanes) {
                const float4 o = *reinterpret_cast<const float4*>(o_s + j * kLdo + col);
                float4 g = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                if (gate) {
                    g = *reinterpret_cast<const float4*>(gate + static_cast<size_t>(j) * p.ld + col);
                    g = make_float4(sigmoid_f(g.x), sigmoid_f(g.y), sigmoid_f(g.z), sigmoid_f(g.w));
                }
                const float n = norm ? 1.0f / sqrtf((ss_s[0][j] + ss_s[1][j]) / static_cast<float>(p.d) + p.eps) : 1.0f;
                *reinterpret_cast<uint2*>(out + static_cast<size_t>(j) * p.H * p.d + col) =
                    make_uint2(pack_bf16(o.x * n * w.x * g.x, o.y * n * w.y * g.y), pack_bf16(o.z * n * w.z * g.z, o.w * n * w.w * g.w));
            }
        }
    } else {
        for (int i = tid; i < a.n * p.d; i += kThreads) {
            const int j = i / p.d, col = i - j * p.d;
            const float n = norm ? norm[col] / sqrtf((ss_s[0][j] + ss_s[1][j]) / static_cast<float>(p.d) + p.eps) : 1.0f;
            out[static_cast<size_t>(j) * p.H * p.d + col] =
                __float2bfloat16_rn(o_s[j * kLdo + col] * n * (gate ? sigmoid_f(gate[static_cast<size_t>(j) * p.ld + col]) : 1.0f));
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------
int width_of(int dim) { return dim <= 64 ? 64 : 128; }

// Chunks of a piece for each sequence: keys, values, sums and images of a piece stay within this many bytes.
constexpr size_t kPieceBytes = 96u << 20;
int chunks_of(const tbl_decay_mixer& m, int n_seq, int n_tok) {
    const size_t units = static_cast<size_t>(n_seq) * m.heads, w = width_of(m.dim);
    const size_t chunk = units * (kTokens * m.dim * 8 + w * w * 6);
    const int all = ceil_div(n_tok, kTokens), most = static_cast<int>(kPieceBytes / chunk);
    return most < 1 ? 1 : (most < all ? most : all);
}

struct Rooms { size_t sums, images, scales, bytes; };
Rooms rooms_of(const tbl_decay_mixer& m, int n_seq, int n_tok) {
    const size_t w = width_of(m.dim), blocks = static_cast<size_t>(n_seq) * m.heads * chunks_of(m, n_seq, n_tok);
    Rooms r{};
    r.sums = 0;
    r.images = round_up(blocks * w * w * 4, 256);
    r.scales = r.images + round_up(blocks * w * w * 2, 256);
    r.bytes = r.scales + round_up(blocks * w * 4, 256);
    return r;
}

template <int DP, int V>
cudaError_t run(ChunkParams c, int per, cudaStream_t st) {
    static bool sums_done[64] = {}, chunk_done[64] = {};
    constexpr size_t sums_smem = 1024 + 6 * (DP / 64) * kBox + (DP == 64 ? kBox : 0);
    constexpr size_t tiles = 3 * (DP / 64) * kSub, collect = sizeof(float) * kTokens * (DP + 4);
    constexpr size_t chunk_smem = 1024 + (tiles > collect ? tiles : collect);
    cudaError_t e = allow_smem(decay_sums_kernel<DP, V>, sums_smem, sums_done);
    if (e == cudaSuccess) e = allow_smem(decay_chunk_kernel<DP, V>, chunk_smem, chunk_done);
    const int units = c.d.n_seq * c.d.H, all = ceil_div(c.d.n_tok, kTokens);
    for (int at = 0; e == cudaSuccess && at < all; at += per) {
        c.first = at * kTokens;
        c.chunks = all - at < per ? all - at : per;
        c.states = at == 0 ? c.d.states : c.d.next;
        e = launch_dependent(decay_sums_kernel<DP, V>, dim3(c.chunks, units), dim3(kThreads), sums_smem, st, c);
        if (e == cudaSuccess) e = launch_dependent(decay_join_kernel<DP>, dim3(DP * DP / 8 / 128, units), dim3(128), 0, st, c);
        if (e == cudaSuccess) e = launch_dependent(decay_chunk_kernel<DP, V>, dim3(c.chunks, units), dim3(kThreads), chunk_smem, st, c);
    }
    return e;
}

}  // namespace

bool decay_chunk_supported(const tbl_decay_mixer& m) { return m.dim <= 128; }

size_t decay_chunk_workspace(const tbl_decay_mixer& m, int n_seq, int n_tok) { return rooms_of(m, n_seq, n_tok).bytes; }

int launch_decay_chunks(const tbl_decay_mixer& m, const DecayParams& p, void* ws, cudaStream_t st) {
    if (static_cast<long long>(p.n_seq) * p.H > 65535) return TBL_ERR_SHAPE;
    const Rooms r = rooms_of(m, p.n_seq, p.n_tok);
    uint8_t* base = static_cast<uint8_t*>(ws);
    ChunkParams c{};
    c.d = p;
    c.sums = reinterpret_cast<float*>(base + r.sums); c.images = base + r.images; c.scales = reinterpret_cast<float*>(base + r.scales);
    const int per = chunks_of(m, p.n_seq, p.n_tok);
    cudaError_t e;
    if (width_of(m.dim) == 64) e = p.vec ? run<64, 4>(c, per, st) : run<64, 1>(c, per, st);
    else e = p.vec ? run<128, 4>(c, per, st) : run<128, 1>(c, per, st);
    return e == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

}  // namespace stack
}  // namespace tbl
