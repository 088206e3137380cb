// Shared by the translation units of the attention over a 4-bit cache (quantized_attention.cu, quantized_decode.cu, quantized_rows.cu).
//
// Cache of a layer: [slot][kv head][token][row], a row being, with n = the head size rounded up to 64, n/2 bytes of key codes, n/2 of value codes,
// n/16 scale bytes of the key, n/16 of the value, and zeros to a multiple of 16.  One token of a head is one contiguous row, so that a tile of tokens
// is one bulk copy.
#pragma once

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "head_rotation.cuh"

namespace tbl {
namespace stack {

__host__ __device__ __forceinline__ int quantized_width(int dim) { return (dim + 63) / 64 * 64; }
__host__ __device__ __forceinline__ int quantized_row(int width) { return (width + width / 8 + 15) / 16 * 16; }

struct QuantizedParams {
    const float* proj;           // [rows][ld]: q | k | v | gate
    const float *q_norm, *k_norm;
    uint8_t* cache;
    const int32_t *slots, *positions;
    void* q;                     // queries, normed and turned: [rows][H][ldq]
    float* q_factor;             // queries in fp16: the power of two they were divided by, [rows][H]
    void* expanded;              // [sequence][kv head][ctx][key | value]: codes x scales, without the layer's units
    float *part_m, *part_l, *part_o;
    void* out;
    int* status;
    Rotation r;
    int ld, g_off;               // of proj; g_off: column of the output gate, < 0: none
    int H, G, group, d, width, row, ldq, ldo, capacity, n_tok, splits, ctx, first_head;    // first_head: of the preparing kernel, H: queries are done already
    float scale_log2, key_unit, value_unit, eps;
};

__device__ __forceinline__ uint8_t* quantized_at(const QuantizedParams& p, int slot, int g, int token) {
    return p.cache + (static_cast<size_t>(slot) * p.G + g) * p.capacity * p.row + static_cast<size_t>(token) * p.row;
}
// a token has room in the cache and, where heads turn, in the tables
__device__ __forceinline__ bool quantized_room(const QuantizedParams& p, int pos) {
    return pos >= 0 && pos < p.capacity && (p.r.half == 0 || pos < p.r.positions);
}

// two codes of a byte (the low half first) as halves
__device__ __forceinline__ __half2 codes_of(uint32_t byte) {
    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(byte), __NV_E2M1);
    return *reinterpret_cast<const __half2*>(&h);
}
__device__ __forceinline__ float scale_of(uint8_t byte) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(byte, __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
}

// Eight numbers of a group of 16, of which the neighbouring lane (lane ^ 1) holds the others: their codes and the group's scale.
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], float unit, uint8_t& scale) {
    float most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        most = fmaxf(most, fabsf(x[i]));
        finite = finite && fabsf(x[i]) < INFINITY;               // false for NaN too
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    finite = (__shfl_xor_sync(0xffffffffu, static_cast<int>(finite), 1) != 0) && finite;
    scale = finite ? __nv_cvt_float_to_fp8(__fdiv_rn(most, __fmul_rn(unit, 6.0f)), __NV_SATFINITE, __NV_E4M3) : 0x7f;
    const float step = __fmul_rn(scale_of(scale), unit);
    uint32_t codes = 0;
    if (!finite || !(step > 0.0f)) return codes;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        codes |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(make_float2(__fdiv_rn(x[2 * i], step), __fdiv_rn(x[2 * i + 1], step)), __NV_E2M1, cudaRoundNearest))
                 << (8 * i);
    return codes;
}

// A head of a row: for a key (turned = its rotation) normed and turned in 64 bits, so that the code of a number does not depend on how a sum of
// squares is rounded; then rounded to 4 bits.  A warp; `mine`: its room for the head's numbers; lane i has the codes of numbers 8 i .. 8 i + 7, even
// lanes the scale of 16.
template <int V>
__device__ __forceinline__ uint32_t quantize_head(const QuantizedParams& p, const float* src, bool is_k, int at, float* mine, int lane, uint8_t& scale) {
    for (int c = p.d + lane; c < p.width; c += 32) mine[c] = 0.0f;
    if (is_k) {
        HeadUnits<V, 32> x;
        x.load(p.r, src, p.d, lane);
        x.template turn<double>(p.r, p.k_norm, p.eps, at, p.d, lane);
        x.store(p.r, mine, p.d, lane);
    } else {
        for (int c = lane; c < p.d; c += 32) mine[c] = src[c];
    }
    __syncwarp();
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = 8 * lane < p.width ? mine[8 * lane + i] : 0.0f;
    const uint32_t codes = quantize8(y, is_k ? p.key_unit : p.value_unit, scale);
    __syncwarp();
    return codes;
}
// its place in a row (in global or shared memory); a value's warp writes the row's padding too
__device__ __forceinline__ void put_row(const QuantizedParams& p, uint8_t* dst, bool is_k, uint32_t codes, uint8_t scale, int lane) {
    if (8 * lane < p.width) {
        reinterpret_cast<uint32_t*>(dst + (is_k ? 0 : p.width / 2))[lane] = codes;
        if ((lane & 1) == 0) dst[p.width + (is_k ? 0 : p.width / 16) + lane / 2] = scale;
    }
    const int used = p.width + p.width / 8;
    if (!is_k && used + lane < p.row) dst[used + lane] = 0;
}
// fp16 queries: the power of two a head is divided by, and the factor that does it
template <int V>
__device__ __forceinline__ float query_power(const HeadUnits<V, 32>& x, float& factor) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < HeadUnits<V, 32>::kUnits; ++i)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) most = fmaxf(most, fabsf(x.x[i][e]));
    const float power = power_of(warp_max(most));
    factor = inverse_power(power) * kUp;
    return power * (1.0f / kUp);
}

// quantized_decode.cu: streams the 4-bit rows for a few query rows
struct StreamPlan {
    int warps, splits;           // of a CTA; of the context
    int most;                    // splits that no shorter context passes (for workspaces)
    int whole;                   // one token of a sequence, no splits: the kernel norms, rounds, appends and finishes by itself
};
int quantized_stream_rows(const tbl_quantized_mixer& m, int n_tok);      // query rows of a CTA
StreamPlan quantized_stream_plan(const tbl_quantized_mixer& m, int n_seq, int n_tok, int context);
int launch_quantized_stream(const QuantizedParams& p, const StreamPlan& plan, int vec, int n_seq, cudaStream_t st);

// quantized_rows.cu: the same in fp32 arithmetic, any number of rows
long long quantized_rows_blocks(const tbl_quantized_mixer& m, int n_seq, int n_tok, int context);     // of query rows
int quantized_rows_splits(const tbl_quantized_mixer& m, int n_seq, int n_tok, int context);
int launch_quantized_rows(const QuantizedParams& p, int precision, int n_seq, cudaStream_t st);

}  // namespace stack
}  // namespace tbl
