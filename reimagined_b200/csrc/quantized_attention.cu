// Softmax attention over a cache that holds keys and values in 4 bits (e2m1 codes, an e4m3 scale for every 16 numbers).
//
//   quantized_prep_kernel    norm and rotation of queries and keys, rounding of keys and values to 4 bits, append
//   quantized_expand_kernel  the visible cache as numbers: code x scale has six bits between 2^-10 and 2688, which fp16 holds
//   quantized_read_kernel    the same for single tokens, in the layer's units
// Prompts go over expanded keys and values through the flash kernel of attention_prefill.cu (in fp16: queries and weights err by 2^-12, down to 2^-25
// of the largest weight, and weights need one term instead of two), a few query rows over the 4-bit rows themselves (quantized_decode.cu), fp32 and
// what else there is in fp32 arithmetic (quantized_rows.cu).  The layer's units enter as factors of the scores and of the output.
#include <math.h>

#include "attention.cuh"
#include "quantized.cuh"

namespace tbl {
namespace stack {
namespace {

constexpr int kPrepWarps = 8;

// A warp per head of a row: query heads, then key heads, then value heads.
template <typename T, int V>
__global__ void __launch_bounds__(32 * kPrepWarps) quantized_prep_kernel(const QuantizedParams p) {
    __shared__ __align__(16) float head_s[kPrepWarps][TBL_MAX_ROTATED_DIM];
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = p.first_head + blockIdx.y * kPrepWarps + warp;
    if (head >= p.H + 2 * p.G) return;
    const int slot = p.slots[row / p.n_tok], pos = p.positions[slot] + row % p.n_tok;
    const bool room = quantized_room(p, pos);
    const int at = p.r.half > 0 ? min(max(pos, 0), p.r.positions - 1) : 0;
    const float* src = p.proj + static_cast<size_t>(row) * p.ld + head * p.d;
    HeadUnits<V, 32> x;
    if (head < p.H) {
        x.load(p.r, src, p.d, lane);
        x.template turn<float>(p.r, p.q_norm, p.eps, at, p.d, lane);
        T* dst = static_cast<T*>(p.q) + (static_cast<size_t>(row) * p.H + head) * p.ldq;
        float f = 1.0f;
        if (sizeof(T) == 2 && p.q_factor) {
            const float power = query_power(x, f);
            if (lane == 0) p.q_factor[static_cast<size_t>(row) * p.H + head] = power;
        }
        x.store(p.r, dst, p.d, lane, f);
        for (int c = p.d + lane; c < p.ldq; c += 32) dst[c] = from_f<T>(0.0f);
        return;
    }
    if (!room) {
        if (head == p.H && lane == 0) atomicOr(p.status, TBL_DEV_CACHE_FULL);
        return;
    }
    const bool is_k = head < p.H + p.G;
    uint8_t scale;
    const uint32_t codes = quantize_head<V>(p, src, is_k, at, head_s[warp], lane, scale);
    put_row(p, quantized_at(p, slot, head - p.H - (is_k ? 0 : p.G), pos), is_k, codes, scale, lane);
}

// ---- cached numbers ---------------------------------------------------------------------------------------------------------
// eight codes times their scale
__device__ __forceinline__ void numbers8(uint32_t codes, float scale, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 c = __half22float2(codes_of((codes >> (8 * i)) & 0xffu));
        v[2 * i] = c.x * scale;
        v[2 * i + 1] = c.y * scale;
    }
}
__device__ __forceinline__ void put8(__half* dst, const float (&v)[8]) {
    __align__(16) __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(h);
}

// [sequence][kv head][ctx][key, padded to 16 | value]; a thread per eight numbers, zeros behind the last visible token.
__global__ void __launch_bounds__(256) quantized_expand_kernel(const QuantizedParams p, const int padded) {
    pdl_launch_dependents();
    pdl_wait();
    const int per = padded / 4;                                  // eights of a row: key and value
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= static_cast<long long>(p.ctx) * per) return;
    const int token = static_cast<int>(i / per), c = static_cast<int>(i % per), is_v = c >= per / 2, e = c - is_v * (per / 2);
    const int seq = blockIdx.y / p.G, g = blockIdx.y % p.G, slot = p.slots[seq];
    const int n = min(p.positions[slot] + p.n_tok, p.capacity);
    float v[8] = {};
    if (token < n) {
        const uint8_t* row = quantized_at(p, slot, g, token);
        const uint32_t codes = reinterpret_cast<const uint32_t*>(row + is_v * (p.width / 2))[e];
        numbers8(codes, scale_of(row[p.width + is_v * (p.width / 16) + e / 2]), v);
    }
    put8(static_cast<__half*>(p.expanded) + ((static_cast<size_t>(blockIdx.y) * p.ctx + token) * per + c) * 8, v);
}

template <typename T>
__global__ void __launch_bounds__(256) quantized_read_kernel(const QuantizedParams p, T* keys, T* values) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x, slot = p.slots[row / p.n_tok], pos = p.positions[slot] + row % p.n_tok, per = p.width / 8;
    if (pos < 0 || pos >= p.capacity) {
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(p.status, TBL_DEV_CACHE_FULL);
        return;
    }
    for (int i = blockIdx.y * 256 + threadIdx.x; i < p.G * 2 * per; i += gridDim.y * 256) {
        const int g = i / (2 * per), c = i - g * 2 * per, is_v = c >= per, e = c - is_v * per;
        T* out = is_v ? values : keys;
        if (!out) continue;
        const uint8_t* src = quantized_at(p, slot, g, pos);
        float v[8];
        numbers8(reinterpret_cast<const uint32_t*>(src + is_v * (p.width / 2))[e], scale_of(src[p.width + is_v * (p.width / 16) + e / 2]), v);
        const float unit = is_v ? p.value_unit : p.key_unit;
        out += (static_cast<size_t>(row) * p.G + g) * p.d + e * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (e * 8 + k < p.d) out[k] = from_f<T>(v[k] * unit);
    }
}

// ---- splits of the context come together --------------------------------------------------------------------------------------
// A CTA per (row, head); a warp takes every eighth split, a lane four neighbouring numbers, so that all partial sums are on their way at once.
constexpr int kMergeWarps = 8;
template <typename T>
__global__ void __launch_bounds__(32 * kMergeWarps) quantized_merge_kernel(const QuantizedParams p) {
    __shared__ __align__(16) float part_s[kMergeWarps][TBL_MAX_ROTATED_DIM];
    pdl_launch_dependents();
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const size_t unit = (static_cast<size_t>(row) * p.H + head) * p.splits;
    pdl_wait();
    const float gate = p.g_off >= 0 && tid < p.d ? p.proj[static_cast<size_t>(row) * p.ld + p.g_off + head * p.d + tid] : 0.0f;
    float most = -INFINITY, sum = 0.0f;
    for (int s = lane; s < p.splits; s += 32) most = fmaxf(most, p.part_m[unit + s]);
    most = warp_max(most);
    for (int s = lane; s < p.splits; s += 32) {
        const float m = p.part_m[unit + s];
        sum = fmaf(p.part_l[unit + s], m == -INFINITY ? 0.0f : ex2(m - most), sum);
    }
    sum = warp_sum(sum);
    float4 acc[TBL_MAX_ROTATED_DIM / 128];
#pragma unroll
    for (int b = 0; b < TBL_MAX_ROTATED_DIM / 128; ++b) acc[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int s = warp; s < p.splits; s += kMergeWarps) {
        const float m = p.part_m[unit + s], f = m == -INFINITY ? 0.0f : ex2(m - most);
        const float* src = p.part_o + (unit + s) * p.ldo;
#pragma unroll
        for (int b = 0; b < TBL_MAX_ROTATED_DIM / 128; ++b)
            if (128 * b + 4 * lane < p.ldo) {
                const float4 x = *reinterpret_cast<const float4*>(src + 128 * b + 4 * lane);
                acc[b].x = fmaf(x.x, f, acc[b].x); acc[b].y = fmaf(x.y, f, acc[b].y); acc[b].z = fmaf(x.z, f, acc[b].z); acc[b].w = fmaf(x.w, f, acc[b].w);
            }
    }
#pragma unroll
    for (int b = 0; b < TBL_MAX_ROTATED_DIM / 128; ++b) *reinterpret_cast<float4*>(&part_s[warp][128 * b + 4 * lane]) = acc[b];
    __syncthreads();
    if (tid < p.d) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) v += part_s[w][tid];
        v *= p.value_unit / sum;
        static_cast<T*>(p.out)[(static_cast<size_t>(row) * p.H + head) * p.d + tid] = from_f<T>(p.g_off >= 0 ? v * sigmoid_f(gate) : v);
    }
}
static_assert(32 * kMergeWarps >= TBL_MAX_ROTATED_DIM, "a thread per number");

// ---- plan -------------------------------------------------------------------------------------------------------------------
enum Route { kAuto = 0, kSimt = 1, kStream = 2, kFlash = 3 };

int padded16(int n) { return static_cast<int>(round_up(n, 16)); }

// the mixer as attention_prefill.cu knows it
tbl_attention_mixer as_attention(const tbl_quantized_mixer& m) {
    tbl_attention_mixer a{};
    a.heads = m.heads; a.kv_heads = m.kv_heads; a.dim = a.vdim = m.dim; a.maps = 1; a.scale = m.scale * m.key_scale; a.kv_from = -1;
    return a;
}

// what the flash kernel's grid and the 32-bit rows of its tensor maps hold (expanded keys and values of every sequence and head, whole blocks of 128)
bool flash_fits(const tbl_quantized_mixer& m, int n_seq, int context) {
    return attention_flash_supported(as_attention(m)) && static_cast<long long>(n_seq) * m.kv_heads * round_up(context, 128) <= 2147483647LL;
}

// bf16: the flash kernel where its time, worked out from what it took, is shorter than the streaming kernel's (32 query and 8 key/value heads of 128,
// in us, streaming and flash kernel: one sequence of 64 tokens over 1024 20 and 43, over 16384 102 and 287; 256 over 4096 115 and 109; 512 over 512 58
// and 45; eight sequences of 64 over 4096 193 and 233, of 128 over 128 86 and 64, over 4096 372 and 244).  Both read or walk the context: the one for
// every block of 8 or 16 query rows, the other a wave of CTAs at a time.
int pick_route(const tbl_quantized_mixer& m, int precision, int n_seq, int n_tok, int context) {
    if (precision != TBL_BF16) return kSimt;
    if (!flash_fits(m, n_seq, context)) return kStream;
    const double rows = static_cast<double>(n_seq) * n_tok, caches = static_cast<double>(n_seq) * m.kv_heads * quantized_width(m.dim) / 128;
    const double seen = context - 0.5 * n_tok, group = m.heads / m.kv_heads;
    const double blocks = ceil(n_tok * group / quantized_stream_rows(m, n_tok));
    const double waves = ceil(n_seq * static_cast<double>(m.heads) * ceil_div(n_tok, 256) / kNumSm);
    const double stream = 11 + 1.8e-3 * rows * m.heads + 42e-6 * caches * blocks * seen * (m.dim > 128 ? 0.7 : 1.0);
    const double flash = 23 + 0.57e-3 * rows * (m.heads + 2 * m.kv_heads) + 250e-6 * caches * context + 0.014 * waves * seen;
    return flash < stream ? kFlash : kStream;
}

struct Plan {
    int route, splits, ctx;
    StreamPlan stream;
    size_t q, factor, expanded, pm, pl, po, bytes;
};

Plan make_plan(const tbl_quantized_mixer& m, int precision, int route, int n_seq, int n_tok, int context) {
    Plan w{};
    const size_t rows = static_cast<size_t>(n_seq) * n_tok, dp = padded16(m.dim);
    w.route = route == kAuto ? pick_route(m, precision, n_seq, n_tok, context) : route;
    w.splits = 1;
    int most = 1;                                                // splits to make room for
    bool parts = w.route == kFlash && !attention_flash_whole(as_attention(m));
    if (w.route == kStream) {
        w.stream = quantized_stream_plan(m, n_seq, n_tok, context);
        w.splits = w.stream.splits;
        most = w.stream.most;
        parts = most > 1;
    } else if (w.route == kSimt) {
        w.splits = most = quantized_rows_splits(m, n_seq, n_tok, context);
        parts = most > 1;
    }
    w.ctx = static_cast<int>(round_up(context, 128));            // whole blocks of the flash kernel
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += round_up(bytes, 256); return at; };
    w.q = take(w.route == kStream ? 2 * rows * m.heads * quantized_width(m.dim) : w.route == kFlash ? 2 * rows * m.heads * dp : 4 * rows * m.heads * m.dim);
    w.factor = take(w.route != kSimt ? sizeof(float) * rows * m.heads : 0);
    w.expanded = take(w.route == kFlash ? 2 * static_cast<size_t>(n_seq) * m.kv_heads * w.ctx * 2 * dp : 0);
    const size_t units = rows * m.heads * most;
    w.pm = take(parts ? sizeof(float) * units : 0);
    w.pl = take(parts ? sizeof(float) * units : 0);
    w.po = take(parts ? sizeof(float) * units * dp : 0);
    w.bytes = off;
    return w;
}

// Bytes of a route.  Without one (0), room for whatever a context no longer than this one takes: a host may ask once for the longest.  (Both times in
// pick_route are straight lines over the context, so the flash kernel is taken somewhere below only if it is at one end.)
size_t bytes_of(const tbl_quantized_mixer& m, int precision, int route, int n_seq, int n_tok, int context) {
    if (route != kAuto || precision != TBL_BF16) return make_plan(m, precision, route, n_seq, n_tok, context).bytes;
    const size_t bytes = make_plan(m, precision, kStream, n_seq, n_tok, context).bytes;
    if (pick_route(m, precision, n_seq, n_tok, n_tok) != kFlash && pick_route(m, precision, n_seq, n_tok, context) != kFlash) return bytes;
    const size_t flash = make_plan(m, precision, kFlash, n_seq, n_tok, context).bytes;
    return bytes > flash ? bytes : flash;
}

template <typename T, int V>
cudaError_t launch_prep_v(const QuantizedParams& p, int rows, cudaStream_t st) {
    return launch_dependent(quantized_prep_kernel<T, V>, dim3(rows, ceil_div(p.H + 2 * p.G - p.first_head, kPrepWarps)), dim3(32 * kPrepWarps), 0, st, p);
}
template <typename T>
cudaError_t launch_prep(const QuantizedParams& p, int rows, bool vec, cudaStream_t st) {
    return vec ? launch_prep_v<T, 4>(p, rows, st) : launch_prep_v<T, 1>(p, rows, st);
}

int launch_merge(const QuantizedParams& p, int precision, int rows, cudaStream_t st) {
    const dim3 grid(rows, p.H), block(32 * kMergeWarps);
    return (precision == TBL_BF16 ? launch_dependent(quantized_merge_kernel<bf16>, grid, block, 0, st, p)
                                  : launch_dependent(quantized_merge_kernel<float>, grid, block, 0, st, p)) == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

int run(const tbl_quantized_mixer& m, int precision, QuantizedParams p, const Plan& w, int n_seq, cudaStream_t st) {
    const int rows = n_seq * p.n_tok;
    // a portion of a prompt: the queries by the kernel that does nothing else (2048 rows of 32 + 16 heads of 128: 51 us all in one)
    if (w.route == kFlash) {
        const RotationCall c{p.proj, p.ld, p.H, 0, p.d, p.slots, p.positions, n_seq, p.n_tok, p.eps, p.q, nullptr, p.q_factor, p.ldq};
        const int rc = launch_head_rotation(m.rotation, precision, c, st);
        if (rc != TBL_OK) return rc;
        p.first_head = p.H;
    }
    const bool vec = vector_heads(m.rotation, p.d, p.proj, p.ld);
    const bool whole = w.route == kStream && w.stream.whole;
    const cudaError_t e = whole ? cudaSuccess : w.route == kSimt ? launch_prep<float>(p, rows, vec, st) : launch_prep<__half>(p, rows, vec, st);
    if (e != cudaSuccess) return TBL_ERR_CUDA;
    if (w.route != kFlash) {
        const int rc = w.route == kStream ? launch_quantized_stream(p, w.stream, vec, n_seq, st) : launch_quantized_rows(p, precision, n_seq, st);
        return rc != TBL_OK || w.splits == 1 ? rc : launch_merge(p, precision, rows, st);
    }
    AttnParams a{};
    a.slots = p.slots; a.positions = p.positions; a.part_m = p.part_m; a.part_l = p.part_l; a.part_o = p.part_o; a.out = p.out; a.status = p.status;
    a.H = p.H; a.G = p.G; a.group = p.group; a.maps = 1; a.d = a.vd = p.d; a.dp = a.vp = padded16(p.d); a.n_tok = p.n_tok; a.splits = 1;
    a.gate = p.g_off < 0 ? nullptr : p.proj + p.g_off; a.ldg = p.ld; a.value_scale = m.value_scale;
    const dim3 grid(ceil_div(static_cast<long long>(p.ctx) * (a.dp / 4), 256), n_seq * p.G);
    if (launch_dependent(quantized_expand_kernel, grid, dim3(256), 0, st, p, a.dp) != cudaSuccess) return TBL_ERR_CUDA;
    a.cache = p.expanded; a.cw = 2 * a.dp; a.n_slots = n_seq; a.capacity = p.ctx; a.by_seq = 1; a.scale_log2 = p.scale_log2;
    a.q16 = static_cast<bf16*>(p.q);                             // sixteen bits either way
    a.q_factor = p.q_factor;
    // the gate's columns decide whether the flash kernel's vector loads are aligned
    a.vec = (p.ld | p.d) % 4 == 0 && aligned16(p.proj);
    const int rc = launch_attention_flash(a, n_seq, st);
    return rc != TBL_OK || attention_flash_whole(as_attention(m)) ? rc : launch_attention_merge(a, precision, rows, st);
}

QuantizedParams basic_params(const tbl_quantized_mixer& m, int capacity, const int32_t* slots, const int32_t* positions, int n_tok) {
    QuantizedParams p{};
    p.slots = slots; p.positions = positions; p.r = rotation_of(m.rotation);
    p.ld = m.in.outputs; p.g_off = m.gated ? (m.heads + 2 * m.kv_heads) * m.dim : -1;
    p.H = m.heads; p.G = m.kv_heads; p.group = m.heads / m.kv_heads; p.d = m.dim; p.width = quantized_width(m.dim); p.row = quantized_row(p.width);
    p.capacity = capacity; p.n_tok = n_tok; p.key_unit = m.key_scale; p.value_unit = m.value_scale;
    p.status = device_status_ptr();
    return p;
}

}  // namespace

int check_quantized(const tbl_quantized_mixer& m, int width) {
    if (m.heads <= 0 || m.kv_heads <= 0 || m.heads > 65535 || m.heads % m.kv_heads) return TBL_ERR_SHAPE;
    const int rc = check_rotation(m.rotation, m.dim);
    if (rc != TBL_OK) return rc;
    auto unit = [](float s) { return s >= 1e-30f && s <= 1e30f; };
    if (!unit(m.key_scale) || !unit(m.value_scale)) return TBL_ERR_SCALE;
    const double factor = static_cast<double>(m.scale) * m.key_scale;       // of the scores: the flash kernel takes their largest before it
    if (!(factor >= 1e-30 && factor <= 1e30)) return TBL_ERR_SCALE;
    if (m.gated != 0 && m.gated != 1) return TBL_ERR_INVALID_ARG;
    const long long cols = (static_cast<long long>(m.heads) * (1 + m.gated) + 2LL * m.kv_heads) * m.dim;
    if (m.in.inputs != width || m.in.outputs != cols || m.out.inputs != m.heads * m.dim || m.out.outputs != width) return TBL_ERR_SHAPE;
    return m.in.weight && m.out.weight ? TBL_OK : TBL_ERR_INVALID_ARG;
}

size_t quantized_slot_bytes(const tbl_quantized_mixer& m, int capacity) {
    return static_cast<size_t>(m.kv_heads) * capacity * quantized_row(quantized_width(m.dim));
}

size_t quantized_workspace(const tbl_quantized_mixer& m, int precision, int n_seq, int n_tok, int context) {
    return bytes_of(m, precision, kAuto, n_seq, n_tok, context);
}

int launch_quantized(const tbl_quantized_mixer& m, int precision, int route, float eps, const float* proj, void* cache, int capacity, const int32_t* slots,
                     const int32_t* positions, int n_seq, int n_tok, int context, void* out, void* ws, cudaStream_t st) {
    const Plan w = make_plan(m, precision, route, n_seq, n_tok, context);
    const long long rows = static_cast<long long>(n_seq) * n_tok;
    if (rows > 2147483647LL || static_cast<long long>(n_seq) * m.kv_heads > 65535 || ceil_div(m.heads + 2 * m.kv_heads, kPrepWarps) > 65535 ||
        w.splits > 65535)
        return TBL_ERR_SHAPE;
    // blocks of query rows are one side of a grid
    const long long total = static_cast<long long>(n_tok) * (m.heads / m.kv_heads), stream_rows = quantized_stream_rows(m, n_tok);
    if ((w.route == kStream && (total + stream_rows - 1) / stream_rows > 65535) ||
        (w.route == kSimt && quantized_rows_blocks(m, n_seq, n_tok, context) > 65535) || (w.route == kFlash && !flash_fits(m, n_seq, context)))
        return TBL_ERR_SHAPE;
    QuantizedParams p = basic_params(m, capacity, slots, positions, n_tok);
    if (!p.status) return TBL_ERR_CUDA;
    uint8_t* base = static_cast<uint8_t*>(ws);
    p.proj = proj; p.q_norm = m.rotation.q_norm; p.k_norm = m.rotation.k_norm; p.cache = static_cast<uint8_t*>(cache); p.out = out; p.eps = eps;
    p.q = base + w.q; p.expanded = base + w.expanded; p.q_factor = w.route != kSimt ? reinterpret_cast<float*>(base + w.factor) : nullptr;
    p.part_m = reinterpret_cast<float*>(base + w.pm); p.part_l = reinterpret_cast<float*>(base + w.pl); p.part_o = reinterpret_cast<float*>(base + w.po);
    p.ldo = padded16(p.d); p.splits = w.splits; p.ctx = w.ctx;
    p.ldq = w.route == kStream ? p.width : w.route == kFlash ? padded16(p.d) : p.d;
    p.scale_log2 = static_cast<float>(static_cast<double>(m.scale) * m.key_scale * 1.4426950408889634);
    return run(m, precision, p, w, n_seq, st);
}

}  // namespace stack
}  // namespace tbl

using namespace tbl;
using namespace tbl::stack;

extern "C" {

int tbl_quantized_row_bytes(const tbl_quantized_mixer* mixer) {
    return mixer && check_quantized(*mixer, mixer->in.inputs) == TBL_OK ? quantized_row(quantized_width(mixer->dim)) : 0;
}

size_t tbl_quantized_workspace_bytes(const tbl_quantized_mixer* mixer, int precision, int route, int n_seq, int n_tok, int context) {
    if (!mixer || (precision != TBL_F32 && precision != TBL_BF16) || route < kAuto || route > kFlash || n_seq <= 0 || n_tok <= 0 || context <= 0 ||
        check_quantized(*mixer, mixer->in.inputs) != TBL_OK)
        return 0;
    return bytes_of(*mixer, precision, route, n_seq, n_tok, context);
}

int tbl_quantized_forward(const tbl_quantized_mixer* mixer, int precision, int route, float eps, const float* proj_dev, void* cache_dev, int slots,
                          int capacity, const int32_t* slots_dev, const int32_t* positions_dev, int n_seq, int n_tok, int context, void* out_dev,
                          void* workspace_dev, size_t workspace_bytes, void* stream) {
    if (!mixer || !proj_dev || !cache_dev || !slots_dev || !positions_dev || !out_dev || n_seq <= 0 || n_tok <= 0 || slots < n_seq || capacity <= 0 ||
        context < n_tok || context > capacity || (precision != TBL_F32 && precision != TBL_BF16) || route < kAuto || route > kFlash || !(eps >= 0.0f))
        return TBL_ERR_INVALID_ARG;
    const int rc = check_quantized(*mixer, mixer->in.inputs);
    if (rc != TBL_OK) return rc;
    if ((route == kStream && precision != TBL_BF16) || (route == kFlash && (precision != TBL_BF16 || !attention_flash_supported(as_attention(*mixer)))))
        return TBL_ERR_SHAPE;
    if (!workspace_dev || workspace_bytes < tbl_quantized_workspace_bytes(mixer, precision, route, n_seq, n_tok, context)) return TBL_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace_dev) & 255) || !aligned16(cache_dev) || !aligned16(out_dev) || (reinterpret_cast<uintptr_t>(proj_dev) & 3))
        return TBL_ERR_ALIGNMENT;
    return launch_quantized(*mixer, precision, route, eps, proj_dev, cache_dev, capacity, slots_dev, positions_dev, n_seq, n_tok, context, out_dev,
                            workspace_dev, static_cast<cudaStream_t>(stream));
}

int tbl_quantized_read(const tbl_quantized_mixer* mixer, int precision, const void* cache_dev, int slots, int capacity, const int32_t* slots_dev,
                       const int32_t* positions_dev, int n_seq, int n_tok, void* keys_dev, void* values_dev, void* stream) {
    if (!mixer || !cache_dev || !slots_dev || !positions_dev || (!keys_dev && !values_dev) || n_seq <= 0 || n_tok <= 0 || slots <= 0 || capacity <= 0 ||
        (precision != TBL_F32 && precision != TBL_BF16))
        return TBL_ERR_INVALID_ARG;
    const int rc = check_quantized(*mixer, mixer->in.inputs);
    if (rc != TBL_OK) return rc;
    const long long rows = static_cast<long long>(n_seq) * n_tok;
    if (rows > 2147483647LL) return TBL_ERR_SHAPE;
    const uintptr_t own = precision == TBL_BF16 ? 1 : 3;
    if (!aligned16(cache_dev) || ((reinterpret_cast<uintptr_t>(keys_dev) | reinterpret_cast<uintptr_t>(values_dev)) & own)) return TBL_ERR_ALIGNMENT;
    QuantizedParams p = basic_params(*mixer, capacity, slots_dev, positions_dev, n_tok);
    if (!p.status) return TBL_ERR_CUDA;
    p.cache = static_cast<uint8_t*>(const_cast<void*>(cache_dev));
    const int most = ceil_div(static_cast<long long>(p.G) * p.width / 4, 256);
    const dim3 grid(static_cast<unsigned>(rows), most < 64 ? most : 64);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto launch = [&](auto kernel, auto* keys, auto* values) { return launch_dependent(kernel, grid, dim3(256), 0, st, p, keys, values); };
    const cudaError_t e = precision == TBL_BF16 ? launch(quantized_read_kernel<bf16>, static_cast<bf16*>(keys_dev), static_cast<bf16*>(values_dev))
                                                : launch(quantized_read_kernel<float>, static_cast<float*>(keys_dev), static_cast<float*>(values_dev));
    return e == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

}  // extern "C"
