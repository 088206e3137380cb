// Linear attention with decay over prompts, by chunks of 128 tokens on the tensor cores (tcgen05).
//
// With y = exp(log_decay) and S the state before a chunk, the token i of the chunk (from 0 on) has
//   o_i = scale (sum_{j <= i} y^(i-j) (q_i . k_j) v_j + y^(i+1) S q_i),      S' = y^n S + sum_j y^(n-1-j) v_j k_j^T.
//
//   decay_sums_kernel    the last sum of every chunk: no chunk waits for another; keys and values as the operands of the products below
//   decay_join_kernel    the states before the chunks one after the other, element by element in fp32
//   decay_chunk_kernel   the outputs of every chunk: two products for the tokens inside, one for the state
// Queries and keys are normed and turned where they are read, from the fp32 projections, which pass through memory once.  A long prompt goes by pieces whose
// operands and sums stay in the second-level cache between the three kernels.
//
// Precision.  The states are sums over the whole sequence and stay fp32: their products take both operands as two fp16 terms each (22 bits, three
// products; numbers 2^-14 below a tile's largest keep fewer).  Outputs are rounded to bf16, so their operands are single fp16 terms under a power of
// two for every token, and for every row of a state: errors of 2^-12.  They are brought up to 2^14, so that numbers down to 2^-28 of the largest
// beside them keep their bits.  A weight y^(i-j) (q_i . k_j) carries the factors of its key and value, and is an fp16 beside the largest weight of
// its row: a token that a row does not see, or has forgotten, takes no bits from it.
#include <cuda_fp16.h>

#include "decay.cuh"
#include "flash.cuh"

namespace tbl {
namespace stack {
namespace {

using namespace tc05;

constexpr int kTokens = 128;
constexpr int kSumThreads = 256, kOutThreads = 512;      // of decay_sums_kernel (its registers would not do for more), of decay_chunk_kernel
constexpr int kSub = 128 * 128;                  // 128 rows of 64 sixteen-bit numbers, 128-byte swizzle
constexpr int kBox = 64 * 128;                   // 64 tokens of the same
constexpr uint32_t kTransposeA = 1u << 15, kTransposeB = 1u << 16;

struct ChunkParams {
    DecayParams d;
    float* sums;                 // [unit][chunk of the piece][key / 4][value][4]
    uint8_t* tokens;             // [unit][chunk]: keys, then values in fp16, as they lie in shared memory (128 rows, swizzled tiles of 64 columns)
    float* powers;               // [unit][chunk][2][128]: the power of two a token's key, value was divided by
    uint8_t* images;             // [unit][chunk]: the state before it as the B operand [value][key] of fp16, as it lies in shared memory
    float* scales;               // [unit][chunk][value]: the power of two its rows were divided by
    const float* states;         // before the piece
    int first, chunks;           // first token of the piece, its chunks for each sequence
    float per_dim;               // 1 / d
};

// sixteen-bit operands that lie with neighbours of the M or N side together: rows of 64 (128 bytes, swizzled), a row per token, groups of 8 tokens 1024 bytes
// apart, the next 64 columns `box` bytes further on
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr, int box) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(box / 16) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// place of column c of row r in tiles of 64 columns, `tile` bytes each
__device__ __forceinline__ uint32_t swizzled(int r, int c, int tile) { return (c >> 6) * tile + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4) + (c & 7) * 2; }

// A head's numbers over the lanes of a warp: LPH lanes for a token, 32 / LPH tokens side by side, eight numbers a lane in units of 2 V
// (head_rotation.cuh).  What does not change from token to token stays in registers: a run's columns, and its place in a row of operands.  EXACT: the
// head is DP wide.
template <int DP, int V, bool EXACT>
struct HeadLane {
    static constexpr int kLph = V == 4 ? DP / 8 : 32, kSide = 32 / kLph, kUnits = 4 / V, kRuns = 2 * kUnits;
    using Units = HeadUnits<V, kLph>;
    int at[kRuns];               // column of a run
    uint32_t mix[kRuns];         // its 16-byte piece of a row of 64, mixed with the lane's own token of those side by side
    __device__ __forceinline__ HeadLane(const Rotation& r, int gl, int group) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) Units::runs(r, gl + kLph * u, at[2 * u], at[2 * u + 1]);
#pragma unroll
        for (int u = 0; u < kRuns; ++u) mix[u] = (((at[u] >> 3) & 7) ^ group) << 4;
    }
    // byte of run u in row k4 + i kSide + group (k4 a multiple of 4) of tiles of 64 columns, `tile` bytes each
    __device__ __forceinline__ uint32_t place(int u, int k4, int i, int group, int tile) const {
        return static_cast<uint32_t>((at[u] >> 6) * tile + (at[u] & 7) * 2 + (k4 + group) * 128) + (mix[u] ^ (((k4 + i * kSide) & 7) << 4)) + i * kSide * 128;
    }
    __device__ __forceinline__ void load(const float* src, int dim, float (&x)[8]) const {
#pragma unroll
        for (int u = 0; u < kRuns; ++u) Units::load_run(src, at[u], EXACT ? 1 << 30 : dim, x + V * u);
    }
    // the angles of a table row for this lane's pairs (units that do not turn: cos 1, sin 0)
    __device__ __forceinline__ void angles(const Rotation& r, int gl, int row, float (&c)[4], float (&s)[4]) const {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int n = V * (gl + kLph * u);
            if (n < r.half) {
                Units::load_run(r.cos + static_cast<size_t>(row) * r.half, n, 1 << 30, c + V * u);
                Units::load_run(r.sin + static_cast<size_t>(row) * r.half, n, 1 << 30, s + V * u);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) { c[V * u + e] = 1.0f; s[V * u + e] = 0.0f; }
            }
        }
    }
    __device__ __forceinline__ void turn(int interleaved, const float (&c)[4], const float (&s)[4], float (&x)[8]) const {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) turn_unit<V>(interleaved, c + V * u, s + V * u, x + 2 * V * u);
    }
};

template <int LPH>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = LPH / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int LPH>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = LPH / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float largest(const float (&x)[8]) {
    float m = fabsf(x[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
    return m;
}
__device__ __forceinline__ float squares(const float (&x)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(x[e], x[e], s);
    return s;
}

__device__ __forceinline__ uint32_t bits_of(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
// V numbers as fp16
template <int V>
__device__ __forceinline__ void put_halves(uint8_t* dst, const float* y) {
    if (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(bits_of(__floats2half2_rn(y[0], y[V > 1 ? 1 : 0])), bits_of(__floats2half2_rn(y[V > 2 ? 2 : 0], y[V > 3 ? 3 : 0])));
    else *reinterpret_cast<__half*>(dst) = __float2half_rn(y[0]);
}
// V numbers as two fp16 terms (22 bits) in tiles `piece` bytes apart, and the first term once more where `also` is
template <int V>
__device__ __forceinline__ void put_terms(uint8_t* dst, int piece, const float* y, uint8_t* also) {
    if (V == 4) {
        const __half2 a = __floats2half2_rn(y[0], y[V > 1 ? 1 : 0]), b = __floats2half2_rn(y[V > 2 ? 2 : 0], y[V > 3 ? 3 : 0]);
        const float2 fa = __half22float2(a), fb = __half22float2(b);
        const uint2 w = make_uint2(bits_of(a), bits_of(b));
        *reinterpret_cast<uint2*>(dst) = w;
        if (also) *reinterpret_cast<uint2*>(also) = w;
        *reinterpret_cast<uint2*>(dst + piece) =
            make_uint2(bits_of(__floats2half2_rn(y[0] - fa.x, y[V > 1 ? 1 : 0] - fa.y)), bits_of(__floats2half2_rn(y[V > 2 ? 2 : 0] - fb.x, y[V > 3 ? 3 : 0] - fb.y)));
    } else {
        const __half a = __float2half_rn(y[0]);
        *reinterpret_cast<__half*>(dst) = a;
        if (also) *reinterpret_cast<__half*>(also) = a;
        *reinterpret_cast<__half*>(dst + piece) = __float2half_rn(y[0] - __half2float(a));
    }
}

struct Place {
    int unit, seq, head, chunk, n, slot, pos0;           // n: tokens of the chunk
    size_t at, row0;                                     // index of (unit, chunk), first row of the projections
};
__device__ __forceinline__ Place place_of(const ChunkParams& c, int unit, int chunk) {
    Place a;
    a.unit = unit; a.seq = unit / c.d.H; a.head = unit % c.d.H; a.chunk = chunk;
    const int first = c.first + chunk * kTokens;
    a.n = min(kTokens, c.d.n_tok - first);
    a.slot = c.d.slots[a.seq];
    a.pos0 = c.d.positions[a.slot] + first;
    a.at = static_cast<size_t>(unit) * c.chunks + chunk;
    a.row0 = static_cast<size_t>(a.seq) * c.d.n_tok + first;
    return a;
}
// Brings rows of 4 d bytes of the projections into the second-level cache for the CTA that will stand where this one does, a wave of two to an SM later: its
// first loads would otherwise wait for memory with nothing else to do.
__device__ __forceinline__ void fetch_ahead(const ChunkParams& c, int column0, int column1) {
    const long long next = static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x + 2 * kNumSm;
    const int unit = static_cast<int>(next / gridDim.x), chunk = static_cast<int>(next % gridDim.x);
    if (unit >= gridDim.y || !c.d.vec || threadIdx.x >= 2 * kTokens) return;
    const int first = c.first + chunk * kTokens, n = min(kTokens, c.d.n_tok - first), j = threadIdx.x % kTokens, column = threadIdx.x < kTokens ? column0 : column1;
    if (j >= n || column < 0) return;
    const float* row = c.d.proj + (static_cast<size_t>(unit / c.d.H) * c.d.n_tok + first + j) * c.d.ld + column + unit % c.d.H * c.d.d;
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row), "r"(c.d.d * 4) : "memory");
}

__device__ __forceinline__ int table_row(const DecayParams& p, int pos) { return p.r.half > 0 ? min(max(pos, 0), p.r.positions - 1) : 0; }

// ---- sums of the chunks -----------------------------------------------------------------------------------------------------------------
// One CTA per (unit, chunk), two tiles of 64 tokens: D[value][key] = sum over a tile's tokens, M = 128 values (of which DP count), N = DP keys; both
// operands lie as they come, a row per token.  Keys are divided by their power of two, values (times the decay to the chunk's end) by the tile's
// largest, both then brought up to 2^14, where fp16 has room below: two terms hold 22 bits, three products 22 bits of the sums, which a tile has in
// columns of its own.  The keys' first terms and the values go to decay_chunk_kernel on the way, as the tiles that it multiplies.  The second tile's
// rows are asked for as soon as the first one's registers are free.  Bound by the way of the rows to the registers (35 % of the issue slots, 40 % of
// the stalls wait for loads); registers and tensor memory leave two CTAs to an SM.  64 chunks of 32 heads: 150 us for 537 MB in and out, 3.6 TB/s.
constexpr float kHighest = 60.0f;                        // (a score of two such heads ends below 2^35)
template <int DP, int V, bool EXACT>
__global__ void __launch_bounds__(kSumThreads, 2) decay_sums_kernel(const ChunkParams c) {
    using Lane = HeadLane<DP, V, EXACT>;
    constexpr int kSumWarps = kSumThreads / 32, kPiece = DP / 64 * kBox, kTile = DP / 64 * kSub, kPerWarp = 64 / kSumWarps;
    constexpr int kRounds = kPerWarp / Lane::kSide, kRuns = Lane::kRuns;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t done;
    __shared__ uint32_t tmem_slot;
    __shared__ float weight_s[kTokens], most_s[2][kSumWarps];       // weight_s: decay from a token to the end of its chunk, 0 behind it
    uint8_t *k_s = smem, *v_s = smem + 2 * kPiece;       // two terms each (the values' last tile may be read past its end: room for that is behind)
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const DecayParams& p = c.d;
    if (tid == 0) {
        mbar_init(&done, 1);
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();                             // (after the allocation: a dependent's would otherwise stand in its way)
    pdl_wait();
    const Place a = place_of(c, blockIdx.y, blockIdx.x);
    fetch_ahead(c, p.H * p.d, p.v_off);
    const float rate = p.log_decay[a.head];
    if (tid < kTokens) weight_s[tid] = tid < a.n - 1 ? expf(rate * static_cast<float>(a.n - 1 - tid)) : tid < a.n ? 1.0f : 0.0f;
    const int group = lane / Lane::kLph, gl = lane % Lane::kLph;
    const Lane kl(p.r, gl, group), vl(Rotation{nullptr, nullptr, 0, 0, 0}, gl, group);
    const float* base = p.proj + a.row0 * p.ld + a.head * p.d;
    if (p.r.half > 0 && tid == 0 && (a.pos0 < 0 || a.pos0 + a.n > p.r.positions)) atomicOr(p.status, TBL_DEV_CACHE_FULL);
    float w[8];
    const bool normed = p.k_norm != nullptr;
    if (normed) kl.load(p.k_norm, p.d, w);
    uint8_t* keys = c.tokens + a.at * 2 * kTile;
    float* powers = c.powers + a.at * 2 * kTokens;
    __syncthreads();
    bool alive = true;
    float back[2];                                       // from a tile's sums to theirs
    float k[kRounds][8], v[kRounds][8];
    // (rows behind the last token: that one again, times 0)
    auto row_of = [&](int tile, int i) { return base + static_cast<size_t>(min(tile * 64 + warp * kPerWarp + group + i * Lane::kSide, a.n - 1)) * p.ld; };
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        kl.load(row_of(0, i) + p.H * p.d, p.d, k[i]);
        vl.load(row_of(0, i) + p.v_off, p.d, v[i]);
    }
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
        float power[kRounds], most = 0.0f;               // power: of two, of a token's key
        const int j0 = tile * 64 + warp * kPerWarp + group;
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int j = j0 + i * Lane::kSide;
            float cs[4], sn[4];
            kl.angles(p.r, gl, table_row(p, a.pos0 + min(j, a.n - 1)), cs, sn);
            if (normed) {
                const float f = rsqrtf(lanes_sum<Lane::kLph>(squares(k[i])) * c.per_dim + p.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) k[i][e] *= w[e] * f;
            }
            kl.turn(p.r.interleaved, cs, sn, k[i]);
            power[i] = power_of(lanes_max<Lane::kLph>(largest(k[i])));
            const float v_most = lanes_max<Lane::kLph>(largest(v[i])), v_power = power_of(v_most);
            most = fmaxf(most, v_most * (weight_s[j] * power[i]));
            // the values as they are, for the products inside the chunk
            const float f = j < a.n ? inverse_power(v_power) * kUp : 0.0f;
#pragma unroll
            for (int u = 0; u < kRuns; ++u) {
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = v[i][V * u + e] * f;
                if (vl.at[u] < DP) put_halves<V>(keys + kTile + vl.place(u, tile * 64 + warp * kPerWarp, i, group, kSub), y);
            }
            if (gl == 0) { powers[j] = power[i]; powers[kTokens + j] = v_power; }
        }
        most = warp_max(most);
        if (lane == 0) most_s[tile][warp] = most;
        if (tile) alive = mbar_wait_bounded(&done, 0, p.status);          // the first tile's products have read their operands
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSumWarps; ++i) most = fmaxf(most, most_s[tile][i]);
        const float top = fmaxf(power_below(most), 7.8886091e-31f), down = inverse_power(top) * kUp;
        back[tile] = top * (1.0f / (kUp * kUp));
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int j = j0 + i * Lane::kSide;
            const float inv = j < a.n ? inverse_power(power[i]) * kUp : 0.0f, f = weight_s[j] * power[i] * down;
#pragma unroll
            for (int u = 0; u < kRuns; ++u) {
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = k[i][V * u + e] * inv;
                if (kl.at[u] < DP)
                    put_terms<V>(k_s + kl.place(u, warp * kPerWarp, i, group, kBox), kPiece, y, keys + kl.place(u, tile * 64 + warp * kPerWarp, i, group, kSub));
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = v[i][V * u + e] * f;
                if (vl.at[u] < DP) put_terms<V>(v_s + vl.place(u, warp * kPerWarp, i, group, kBox), kPiece, y, nullptr);
            }
            if (tile == 0) {                             // these registers are free: the second tile's numbers come under what is left of the first
                kl.load(row_of(1, i) + p.H * p.d, p.d, k[i]);
                vl.load(row_of(1, i) + p.v_off, p.d, v[i]);
            }
        }
        fence_proxy_async();
        __syncthreads();
        if (warp == 0 && elect_one() && alive) {
            tc_fence_after();
            const uint32_t id = idesc_f16(DP) | kTransposeA | kTransposeB, d = tmem + tile * DP;
            const uint64_t vd = desc_rows(smem_u32(v_s), kBox), kd = desc_rows(smem_u32(k_s), kBox);
            constexpr int kStep = kPiece / 16;
#pragma unroll
            for (int s = 0; s < 4; ++s) {                // the small products first, 16 tokens each
                umma_f16(d, vd + kStep + 128 * s, kd + 128 * s, id, s != 0);
                umma_f16(d, vd + 128 * s, kd + kStep + 128 * s, id, 1);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) umma_f16(d, vd + 128 * s, kd + 128 * s, id, 1);
            umma_commit(&done);
        }
    }
    alive = mbar_wait_bounded(&done, 1, p.status) && alive;
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;              // value
    if (alive && (warp & 3) * 32 < DP) {
        float* dst = c.sums + a.at * DP * DP;
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
                f.x = fmaf(__uint_as_float(x[e]), back[0], __uint_as_float(y[e]) * back[1]);
                f.y = fmaf(__uint_as_float(x[e + 1]), back[0], __uint_as_float(y[e + 1]) * back[1]);
                f.z = fmaf(__uint_as_float(x[e + 2]), back[0], __uint_as_float(y[e + 2]) * back[1]);
                f.w = fmaf(__uint_as_float(x[e + 3]), back[0], __uint_as_float(y[e + 3]) * back[1]);
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
// DP / 8 lanes share a row (a value's keys), eight neighbouring keys each; the next eight chunks' sums are on their way.  64 chunks of 32 heads: 53
// us for 201 MB.
template <int DP>
__global__ void __launch_bounds__(128) decay_join_kernel(const ChunkParams c) {
    constexpr int kLph = DP / 8, kSide = 32 / kLph;
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
    constexpr int kAhead = 8;
    float4 x[kAhead][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < c.chunks) { x[i][0] = src[static_cast<size_t>(i) * DP * DP / 4]; x[i][1] = src[static_cast<size_t>(i) * DP * DP / 4 + DP]; }
    const Decay whole(rate * static_cast<float>(kTokens));
    for (int i0 = 0; i0 < c.chunks; i0 += kAhead) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k;
            if (i >= c.chunks) break;
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(s[e]));
            most = lanes_max<kLph>(most);
            const float power = power_of(most), inv = inverse_power(power) * kUp;
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
            const Decay l = n == kTokens ? whole : Decay(rate * static_cast<float>(n));
            const float4 u = x[k][0], v = x[k][1];
            s[0] = l.of(s[0]) + u.x; s[1] = l.of(s[1]) + u.y; s[2] = l.of(s[2]) + u.z; s[3] = l.of(s[3]) + u.w;
            s[4] = l.of(s[4]) + v.x; s[5] = l.of(s[5]) + v.y; s[6] = l.of(s[6]) + v.z; s[7] = l.of(s[7]) + v.w;
            if (i + kAhead < c.chunks) {
                x[k][0] = src[static_cast<size_t>(i + kAhead) * DP * DP / 4];
                x[k][1] = src[static_cast<size_t>(i + kAhead) * DP * DP / 4 + DP];
            }
        }
    }
    // (only now: CTAs of the next kernel that come early find room on few SMs, two to one, and stay there; 32 heads, 128 tokens 26 to 31 us as it
    // fell out and 26 so, 512 tokens 38 and 30)
    pdl_launch_dependents();
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (row < p.d && 8 * gl + e < p.d) p.next[state + 8 * gl + e] = s[e];
}

// ---- outputs of the chunks ----------------------------------------------------------------------------------------------------------------
// One CTA per (unit, chunk).  Scores Q K^T in the first 128 columns of its tensor memory, weights in their place (fp16, the A operand of the second
// product), the tokens' part of the outputs behind them, then the state's part over the weights.  Keys and values come by bulk copies while the
// queries are normed, the state's operand by another into the keys' room.  Outputs are collected in shared memory, so that gates are read and rows
// are written whole.  512 threads, since it is their loads and barriers that take the time (44 % of the issue slots; with 256 threads 174 instead of
// 163 us): 64 chunks of 32 heads 160 us for 537 MB, 3.4 TB/s.
template <int DP, int V, bool EXACT>
__global__ void __launch_bounds__(kOutThreads, 2) decay_chunk_kernel(const ChunkParams c) {
    using Lane = HeadLane<DP, V, EXACT>;
    constexpr int kTile = DP / 64 * kSub, kPerWarp = kTokens / (kOutThreads / 32), kLdo = DP + 4, kImage = DP * DP * 2;
    constexpr int kRounds = kPerWarp / Lane::kSide, kFlight = kRounds < 2 ? kRounds : 2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(16) float kv_f[kTokens], scale_s[DP];
    __shared__ float power_s[kTokens + 1], q_f[kTokens], ss_s[4][kTokens], most_s;       // power_s: y^n; ss_s: first the weights' maxima, then sums of squares
    __shared__ __align__(8) uint64_t bars[4];            // keys and values, scores, state's image, outputs
    __shared__ uint32_t tmem_slot;
    uint8_t *q_s = smem, *k_s = smem + kTile, *v_s = smem + 2 * kTile;
    float* o_s = reinterpret_cast<float*>(smem);         // afterwards: [token][kLdo]
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const DecayParams& p = c.d;
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) mbar_init(&bars[i], 1);
        fence_mbar_init();
        fence_proxy_async();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();
    const Place a = place_of(c, blockIdx.y, blockIdx.x);
    if (warp == 0 && elect_one()) {
        mbar_arrive_expect_tx(&bars[0], 2 * kTile);
        bulk_g2s(k_s, c.tokens + a.at * 2 * kTile, 2 * kTile, &bars[0]);
    }
    __syncwarp();
    fetch_ahead(c, 0, p.g_off);
    const float rate = p.log_decay[a.head];
    if (tid <= kTokens) power_s[tid] = tid ? expf(rate * static_cast<float>(tid)) : 1.0f;
    if (tid < DP) scale_s[tid] = c.scales[a.at * DP + tid];
    const int group = lane / Lane::kLph, gl = lane % Lane::kLph;
    const float* base = p.proj + a.row0 * p.ld + a.head * p.d;
    {
        const Lane ql(p.r, gl, group);
        float w[8];
        const bool normed = p.q_norm != nullptr;
        if (normed) ql.load(p.q_norm, p.d, w);
#pragma unroll 1
        for (int i0 = 0; i0 < kRounds; i0 += kFlight) {
            float x[kFlight][8];
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const int j = warp * kPerWarp + (i0 + i) * Lane::kSide + group;
                ql.load(base + static_cast<size_t>(min(j, a.n - 1)) * p.ld, p.d, x[i]);
            }
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const int j = warp * kPerWarp + (i0 + i) * Lane::kSide + group;
                float cs[4], sn[4];
                ql.angles(p.r, gl, table_row(p, a.pos0 + min(j, a.n - 1)), cs, sn);
                if (normed) {
                    const float inv = rsqrtf(lanes_sum<Lane::kLph>(squares(x[i])) * c.per_dim + p.eps);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][e] *= w[e] * inv;
                }
                ql.turn(p.r.interleaved, cs, sn, x[i]);
                const float power = power_of(lanes_max<Lane::kLph>(largest(x[i]))), f = inverse_power(power) * kUp;
#pragma unroll
                for (int u = 0; u < Lane::kRuns; ++u) {
                    float y[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) y[e] = x[i][V * u + e] * f;
                    if (ql.at[u] < DP) put_halves<V>(q_s + ql.place(u, warp * kPerWarp, i0 + i, group, kSub), y);
                }
                if (gl == 0) q_f[j] = power;
            }
        }
    }
    fence_proxy_async();
    __syncthreads();
    bool alive = true;
    if (warp == 0) {
        if (elect_one()) {
            const bool there = mbar_wait_bounded(&bars[0], 0, p.status);
            tc_fence_after();
            if (there) flash::products(tmem, smem_desc_sw128(smem_u32(q_s)), smem_desc_sw128(smem_u32(k_s)), DP / 16, idesc_f16(kTokens), 0);
            umma_commit(&bars[1]);
        }
        __syncwarp();
    } else if (warp == 1) {                              // the factors of a token's key and value together, 2^kHighest for the largest
        const float* powers = c.powers + a.at * 2 * kTokens;
        float f[kTokens / 32], most = -254.0f;
#pragma unroll
        for (int i = 0; i < kTokens / 32; ++i) {
            const int j = lane + 32 * i;
            // (as exponents: the product of two powers of two may pass the ends of fp32)
            f[i] = static_cast<float>(static_cast<int>(__float_as_uint(powers[j]) >> 23) + static_cast<int>(__float_as_uint(powers[kTokens + j]) >> 23) - 254);
            if (j < a.n) most = fmaxf(most, f[i]);
        }
        most = warp_max(most);
#pragma unroll
        for (int i = 0; i < kTokens / 32; ++i) kv_f[lane + 32 * i] = lane + 32 * i < a.n ? exp2f(f[i] - most + kHighest) : 0.0f;
        if (lane == 0) most_s = most;
    }
    __syncthreads();
    alive = mbar_wait_bounded(&bars[1], 0, p.status);
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    if (alive && warp == 0 && elect_one()) {             // the keys are done with
        mbar_arrive_expect_tx(&bars[2], kImage);
        bulk_g2s(k_s, c.images + a.at * kImage, kImage, &bars[2]);
    }
    __syncwarp();
    const int row = (warp & 3) * 32 + lane, ch = warp >> 2;          // a thread has a row's fourth
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float row_power;                                     // of the row's largest weight
    {
        uint32_t x[32];
        float most = 0.0f;
        if (ch <= (warp & 3)) {                          // otherwise nothing of it is visible to these rows
            tmem_ld32(tmem + lanes + ch * 32, x);
            tmem_ld_wait();
            const float* power = power_s + (row - ch * 32);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                const float4 f4 = *reinterpret_cast<const float4*>(kv_f + ch * 32 + e);
                const float f[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool seen = ch < (warp & 3) || e + k <= lane;
                    const float w = seen ? __uint_as_float(x[e + k]) * power[-(seen ? e + k : 0)] * f[k] : 0.0f;
                    most = fmaxf(most, fabsf(w));
                    x[e + k] = __float_as_uint(w);
                }
            }
        }
        ss_s[ch][row] = most;
        asm volatile("bar.sync %0, 128;" ::"r"(1 + (warp & 3)) : "memory");           // the four warps that share these rows
        row_power = power_of(fmaxf(fmaxf(ss_s[0][row], ss_s[1][row]), fmaxf(ss_s[2][row], ss_s[3][row])));
        const float f = inverse_power(row_power) * kUp;
        uint32_t y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
            y[e] = ch <= (warp & 3) ? bits_of(__floats2half2_rn(__uint_as_float(x[2 * e]) * f, __uint_as_float(x[2 * e + 1]) * f)) : 0u;
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
        const bool image = mbar_wait_bounded(&bars[2], 0, p.status);
        if (image) flash::products(tmem, smem_desc_sw128(smem_u32(q_s)), smem_desc_sw128(smem_u32(k_s)), DP / 16, idesc_f16(DP), 0);
        umma_commit(&bars[3]);
    }
    __syncwarp();
    if (alive) alive = mbar_wait_bounded(&bars[3], 0, p.status);
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    // the sums of squares of a row's fourths meet in shared memory
    const float row_bits = static_cast<float>(static_cast<int>(__float_as_uint(row_power) >> 23) - 127);
    const float f = q_f[row] * p.scale, inside = f * exp2f(most_s + row_bits - (kHighest + 4 * kUpBits));
    const float before = f * power_s[min(row + 1, kTokens)] * (1.0f / (kUp * kUp));
    float ss = 0.0f;
#pragma unroll 1
    for (int q = 0; q < DP / 64; ++q) {
        const int col = ch * (DP / 4) + 16 * q;
        uint32_t x[16], y[16];
        tmem_ld16(tmem + lanes + kTokens + col, x);
        tmem_ld16(tmem + lanes + col, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4 g = *reinterpret_cast<const float4*>(scale_s + col + e);
            float4 o;                                    // (columns from d on are zeros)
            o.x = fmaf(__uint_as_float(x[e]), inside, __uint_as_float(y[e]) * (before * g.x));
            o.y = fmaf(__uint_as_float(x[e + 1]), inside, __uint_as_float(y[e + 1]) * (before * g.y));
            o.z = fmaf(__uint_as_float(x[e + 2]), inside, __uint_as_float(y[e + 2]) * (before * g.z));
            o.w = fmaf(__uint_as_float(x[e + 3]), inside, __uint_as_float(y[e + 3]) * (before * g.w));
            ss = fmaf(o.x, o.x, ss); ss = fmaf(o.y, o.y, ss); ss = fmaf(o.z, o.z, ss); ss = fmaf(o.w, o.w, ss);
            *reinterpret_cast<float4*>(o_s + row * kLdo + col + e) = o;
        }
    }
    ss_s[ch][row] = ss;
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
    }
    if (!alive) return;
    bf16* out = static_cast<bf16*>(p.out) + (a.row0 * p.H + a.head) * p.d;
    const float* gate = p.g_off < 0 ? nullptr : base + p.g_off;
    const float* norm = p.norm ? p.norm + a.head * p.d : nullptr;
    const bool vec = p.vec && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 && (reinterpret_cast<uintptr_t>(p.norm) & 15) == 0;
    // (the gate's sigmoid by the fast exponential and reciprocal, 2^-21 each, before a rounding of 2^-9)
    auto open = [](float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); };
    auto row_factor = [&](int j) { return norm ? rsqrtf(((ss_s[0][j] + ss_s[1][j]) + (ss_s[2][j] + ss_s[3][j])) * c.per_dim + p.eps) : 1.0f; };
    if (vec) {
        constexpr int kLanes = DP / 4, kRows = kOutThreads / kLanes, kBatch = 4;            // lanes to a row, rows at a time
        const int col = (tid % kLanes) * 4, j0 = tid / kLanes;
        if (col >= p.d) return;
        float4 w = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (norm) w = *reinterpret_cast<const float4*>(norm + col);
#pragma unroll 1
        for (int b = 0; b < kTokens / kRows; b += kBatch) {
            float4 g[kBatch];
            if (gate) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    g[i] = *reinterpret_cast<const float4*>(gate + static_cast<size_t>(min(j0 + (b + i) * kRows, a.n - 1)) * p.ld + col);
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int j = j0 + (b + i) * kRows;
                if (j >= a.n) continue;
                float4 o = *reinterpret_cast<const float4*>(o_s + j * kLdo + col);
                const float n = row_factor(j);
                o = make_float4(o.x * n * w.x, o.y * n * w.y, o.z * n * w.z, o.w * n * w.w);
                if (gate) o = make_float4(o.x * open(g[i].x), o.y * open(g[i].y), o.z * open(g[i].z), o.w * open(g[i].w));
                *reinterpret_cast<uint2*>(out + static_cast<size_t>(j) * p.H * p.d + col) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
            }
        }
    } else {
        for (int i = tid; i < a.n * p.d; i += kOutThreads) {
            const int j = i / p.d, col = i - j * p.d;
            out[static_cast<size_t>(j) * p.H * p.d + col] = __float2bfloat16_rn(o_s[j * kLdo + col] * row_factor(j) * (norm ? norm[col] : 1.0f) *
                                                                                (gate ? open(gate[static_cast<size_t>(j) * p.ld + col]) : 1.0f));
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------
int width_of(int dim) { return dim <= 64 ? 64 : 128; }

// Chunks of a piece for each sequence: keys, values and what is made of them stay within this many bytes, and the two large kernels' last CTAs fill
// the GPU (8192 tokens of 32 heads, before weights had their row's maximum, which costs 2 us: pieces of 9, 18, 37 and 64 chunks take 433, 414, 404 and 411 us,
// 39 chunks 418).
constexpr size_t kPieceBytes = 352u << 20;
int most_chunks(const tbl_decay_mixer& m, int n_seq, int n_tok) {
    const size_t w = width_of(m.dim), chunk = static_cast<size_t>(n_seq) * m.heads * (kTokens * (m.dim * 8 + w * 4) + w * w * 6), most = kPieceBytes / chunk;
    const int all = ceil_div(n_tok, kTokens);
    return most >= static_cast<size_t>(all) ? all : most ? static_cast<int>(most) : 1;
}
int chunks_of(const tbl_decay_mixer& m, int n_seq, int n_tok) {
    const int most = most_chunks(m, n_seq, n_tok);
    if (most == ceil_div(n_tok, kTokens)) return most;
    const size_t units = static_cast<size_t>(n_seq) * m.heads, wave = 2 * kNumSm, full = units * most / wave * wave / units;
    return full ? static_cast<int>(full) : most;
}

struct Rooms { size_t sums, tokens, powers, images, scales, bytes; };
Rooms rooms_of(const tbl_decay_mixer& m, int n_seq, int n_tok) {
    const size_t w = width_of(m.dim), blocks = static_cast<size_t>(n_seq) * m.heads * most_chunks(m, n_seq, n_tok);
    Rooms r{};
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += round_up(bytes, 256); return at; };
    r.sums = take(blocks * w * w * 4);
    r.tokens = take(blocks * kTokens * w * 4);
    r.powers = take(blocks * kTokens * 8);
    r.images = take(blocks * w * w * 2);
    r.scales = take(blocks * w * 4);
    r.bytes = off;
    return r;
}

template <int DP, int V, bool EXACT>
cudaError_t run(ChunkParams c, int per, cudaStream_t st) {
    static bool sums_done[64] = {}, chunk_done[64] = {};
    constexpr size_t sums_smem = 1024 + 4 * (DP / 64) * kBox + (DP == 64 ? kBox : 0);
    constexpr size_t tiles = 3 * (DP / 64) * kSub, collect = sizeof(float) * kTokens * (DP + 4);
    constexpr size_t chunk_smem = 1024 + (tiles > collect ? tiles : collect);
    cudaError_t e = allow_smem(decay_sums_kernel<DP, V, EXACT>, sums_smem, sums_done);
    if (e == cudaSuccess) e = allow_smem(decay_chunk_kernel<DP, V, EXACT>, chunk_smem, chunk_done);
    const int units = c.d.n_seq * c.d.H, all = ceil_div(c.d.n_tok, kTokens);
    for (int at = 0; e == cudaSuccess && at < all; at += per) {
        c.first = at * kTokens;
        c.chunks = all - at < per ? all - at : per;
        c.states = at == 0 ? c.d.states : c.d.next;
        e = launch_dependent(decay_sums_kernel<DP, V, EXACT>, dim3(c.chunks, units), dim3(kSumThreads), sums_smem, st, c);
        if (e == cudaSuccess) e = launch_dependent(decay_join_kernel<DP>, dim3(DP * DP / 8 / 128, units), dim3(128), 0, st, c);
        if (e == cudaSuccess) e = launch_dependent(decay_chunk_kernel<DP, V, EXACT>, dim3(c.chunks, units), dim3(kOutThreads), chunk_smem, st, c);
    }
    return e;
}
template <int DP>
cudaError_t run_width(const ChunkParams& c, int per, cudaStream_t st) {
    if (!c.d.vec) return run<DP, 1, false>(c, per, st);
    return c.d.d == DP ? run<DP, 4, true>(c, per, st) : run<DP, 4, false>(c, per, st);
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
    c.per_dim = 1.0f / static_cast<float>(p.d);
    c.sums = reinterpret_cast<float*>(base + r.sums); c.tokens = base + r.tokens; c.powers = reinterpret_cast<float*>(base + r.powers);
    c.images = base + r.images; c.scales = reinterpret_cast<float*>(base + r.scales);
    const int per = chunks_of(m, p.n_seq, p.n_tok);
    const cudaError_t e = width_of(m.dim) == 64 ? run_width<64>(c, per, st) : run_width<128>(c, per, st);
    return e == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

}  // namespace stack
}  // namespace tbl
