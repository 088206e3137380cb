// Shared by the translation units of linear attention with decay (decay_attention.cu, decay_chunk.cu).
#pragma once

#include "head_rotation.cuh"

namespace tbl {
namespace stack {

struct DecayParams {
    const float* proj;           // [rows][ld]: q | k | v | gate
    const float *q, *k;          // scan: normed and turned, [rows][H][d]
    float* raw;                  // scan: scale S q, [rows][H][d]
    float* starts;               // scan by segments: the states before them, [unit][segment][value][key]
    const float *log_decay, *norm;
    const float* states;         // [slots][H][value][key]
    float* next;                 // the same, after the last token
    const int32_t *slots, *positions;
    void* out;                   // [rows][H * d]
    int* status;
    Rotation r;
    const float *q_norm, *k_norm;
    int ld, H, d, v_off, g_off, n_seq, n_tok, vec, segments, segment;          // segments of `segment` tokens, the last one what is left
    float scale, eps;
};

// What exp(log_decay) -- or several tokens' together, exp(log) -- leaves of a state s: m s + (slow ? s : 0).  A slow decay enters as 1 - exp(log),
// which has 24 bits however slow it is, whereas a decay rounded to fp32 would be off by 2^-25 every token, all in one direction; a fast one as
// itself, which has 24 bits however little it leaves, whereas 1 - exp(log) would be off by 2^-25 of the state before (as much
// as is left of it after 17 in the exponent).  Where it is a token's the loops are there twice: a scan of 3 x 301 tokens 58.4 -> 59.4 us.
struct Decay {
    float m;
    bool slow;
    __device__ __forceinline__ explicit Decay(float log) : slow(log > -0.5f) { m = slow ? expm1f(log) : expf(log); }
    __device__ __forceinline__ float of(float s) const { return fmaf(m, s, slow ? s : 0.0f); }
};

// decay_chunk.cu: prompts by chunks on the tensor cores
bool decay_chunk_supported(const tbl_decay_mixer& m);
size_t decay_chunk_workspace(const tbl_decay_mixer& m, int n_seq, int n_tok);
int launch_decay_chunks(const tbl_decay_mixer& m, const DecayParams& p, void* ws, cudaStream_t st);

}  // namespace stack
}  // namespace tbl
