// Norm and rotation of query and key heads (tbl_head_rotation), shared by the operator of its own (head_rotation.cu) and the mixers that
// open with it.
#pragma once

#include <cuda_fp16.h>
#include <string.h>

#include "stack.cuh"

namespace tbl {
namespace stack {

template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

struct Rotation {
    const float *cos, *sin;      // [positions][half]
    int half, positions, interleaved;
};
inline Rotation rotation_of(const tbl_head_rotation& r) { return Rotation{r.rope_cos, r.rope_sin, r.rot_dim / 2, r.rope_positions, r.interleaved}; }

__device__ __forceinline__ float reciprocal_root(float v) { return rsqrtf(v); }          // 2 units in the last place
__device__ __forceinline__ double reciprocal_root(double v) { return 1.0 / sqrt(v); }

// The V pairs of a unit y [2 V] turn by their cosines and sines: the two runs of V, or neighbours.
template <int V, typename A>
__device__ __forceinline__ void turn_unit(int interleaved, const float* c, const float* s, A* y) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (interleaved) {
            const A p = y[2 * j], q = y[2 * j + 1];
            y[2 * j] = p * A(c[j]) - q * A(s[j]);
            y[2 * j + 1] = q * A(c[j]) + p * A(s[j]);
        } else {
            const A p = y[j], q = y[V + j];
            y[j] = p * A(c[j]) - q * A(s[j]);
            y[V + j] = q * A(c[j]) + p * A(s[j]);
        }
    }
}

// A head spread over LPH lanes, in units of 2 V numbers: V pairs (a, b) that turn together, or numbers that do not turn.  Without `interleaved` a
// unit that turns is two runs of V neighbours half a rotated part apart, otherwise it is 2 V neighbours.  V = 4: 16-byte accesses (vector_heads
// below), V = 2: 8-byte ones (paired_heads), V = 1: any size.
template <int V, int LPH>
struct HeadUnits {
    static constexpr int kUnits = V == 4 ? 1 : TBL_MAX_ROTATED_DIM / (2 * V) / LPH;      // vectors: callers choose LPH >= dim / 8
    float x[kUnits][2 * V];

    // where unit u begins, and its second run of V numbers
    static __device__ __forceinline__ void runs(const Rotation& r, int u, int& a, int& b) {
        const int turning = r.half / V;
        a = u < turning ? (r.interleaved ? 2 * V * u : V * u) : 2 * r.half + 2 * V * (u - turning);
        b = u < turning && !r.interleaved ? a + r.half : a + V;
    }
    static __device__ __forceinline__ void load_run(const float* src, int at, int dim, float* v) {
        if (V == 4) {
            const float4 f = at < dim ? *reinterpret_cast<const float4*>(src + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v[0] = f.x; v[V > 1 ? 1 : 0] = f.y; v[V > 2 ? 2 : 0] = f.z; v[V > 3 ? 3 : 0] = f.w;
        } else if (V == 2) {
            const float2 f = at < dim ? *reinterpret_cast<const float2*>(src + at) : make_float2(0.0f, 0.0f);
            v[0] = f.x; v[V > 1 ? 1 : 0] = f.y;
        } else {
            v[0] = at < dim ? src[at] : 0.0f;
        }
    }
    __device__ __forceinline__ void load(const Rotation& r, const float* src, int dim, int lane) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            int a, b;
            runs(r, lane + LPH * i, a, b);
            load_run(src, a, dim, x[i]);
            load_run(src, b, dim, x[i] + V);
        }
    }
    // Norm (weight null: none) and rotation by the tables' row `pos`, worked out in A.
    template <typename A>
    __device__ __forceinline__ void turn(const Rotation& r, const float* weight, float eps, int pos, int dim, int lane) {
        A inv = A(1);
        if (weight) {
            A ss = A(0);
#pragma unroll
            for (int i = 0; i < kUnits; ++i)
#pragma unroll
                for (int e = 0; e < 2 * V; ++e) ss += A(x[i][e]) * A(x[i][e]);
#pragma unroll
            for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = reciprocal_root(ss / A(dim) + A(eps));
        }
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = lane + LPH * i;
            int a, b;
            runs(r, u, a, b);
            A y[2 * V];
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) y[e] = A(x[i][e]);
            if (weight) {
                float w[2 * V];
                load_run(weight, a, dim, w);
                load_run(weight, b, dim, w + V);
#pragma unroll
                for (int e = 0; e < 2 * V; ++e) y[e] = y[e] * inv * A(w[e]);
            }
            if (u < r.half / V) {
                float c[V], s[V];
                load_run(r.cos + static_cast<size_t>(pos) * r.half, V * u, r.half, c);
                load_run(r.sin + static_cast<size_t>(pos) * r.half, V * u, r.half, s);
                turn_unit<V>(r.interleaved, c, s, y);
            }
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) x[i][e] = static_cast<float>(y[e]);
        }
    }
    template <typename T>
    static __device__ __forceinline__ void store_run(T* dst, int at, int dim, const float* v, float f) {
        if (at >= dim) return;
        if (V == 4 && sizeof(T) == 4) {
            *reinterpret_cast<float4*>(dst + at) = make_float4(v[0] * f, v[V > 1 ? 1 : 0] * f, v[V > 2 ? 2 : 0] * f, v[V > 3 ? 3 : 0] * f);
        } else if (V == 4) {
            T t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = from_f<T>(v[V > 1 ? e : 0] * f);
            uint2 w;
            memcpy(&w, t, sizeof(w) < sizeof(t) ? sizeof(w) : sizeof(t));
            *reinterpret_cast<uint2*>(dst + at) = w;
        } else if (V == 2 && sizeof(T) == 4) {
            *reinterpret_cast<float2*>(dst + at) = make_float2(v[0] * f, v[V > 1 ? 1 : 0] * f);
        } else if (V == 2) {
            T t[2] = {from_f<T>(v[0] * f), from_f<T>(v[V > 1 ? 1 : 0] * f)};
            uint32_t w;
            memcpy(&w, t, sizeof(w) < sizeof(t) ? sizeof(w) : sizeof(t));
            *reinterpret_cast<uint32_t*>(dst + at) = w;
        } else {
            dst[at] = from_f<T>(v[0] * f);
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(const Rotation& r, T* dst, int dim, int lane, float f = 1.0f) const {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            int a, b;
            runs(r, lane + LPH * i, a, b);
            store_run(dst, a, dim, x[i], f);
            store_run(dst, b, dim, x[i] + V, f);
        }
    }
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// whether runs of four numbers of every head, weight and table lie on 16 bytes
inline bool vector_heads(const tbl_head_rotation& r, int dim, const void* proj, int ld) {
    const int half = r.rot_dim / 2;
    return dim % 8 == 0 && half % 4 == 0 && ld % 4 == 0 && aligned16(proj) && aligned16(r.q_norm) && aligned16(r.k_norm) && aligned16(r.rope_cos) &&
           aligned16(r.rope_sin);
}

// whether runs of two do (the last unit of four numbers may have only its first run)
inline bool paired_heads(const tbl_head_rotation& r, int dim, const void* proj, int ld, const void* q, const void* k) {
    auto on8 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; };
    return dim % 2 == 0 && r.rot_dim % 4 == 0 && ld % 2 == 0 && on8(proj) && on8(r.q_norm) && on8(r.k_norm) && on8(r.rope_cos) && on8(r.rope_sin) && on8(q) && on8(k);
}

inline int check_rotation(const tbl_head_rotation& r, int dim) {
    if (dim <= 0 || dim > TBL_MAX_ROTATED_DIM || r.rot_dim < 0 || r.rot_dim > dim || r.rot_dim % 2) return TBL_ERR_SHAPE;
    if (r.interleaved != 0 && r.interleaved != 1) return TBL_ERR_INVALID_ARG;
    if (r.rot_dim > 0 && (!r.rope_cos || !r.rope_sin || r.rope_positions <= 0)) return TBL_ERR_INVALID_ARG;
    return TBL_OK;
}

// the power of two at or below v (1 for 0)
__device__ __forceinline__ float power_below(float v) {
    const uint32_t power = min(__float_as_uint(v) >> 23, 253u);
    return power ? __uint_as_float(power << 23) : 1.0f;
}
// Numbers as fp16: under the power of two at or below the largest of them (2^-113 at least, also for zeros, which so count less than anything else),
// and brought up by kUp to below 2^14, so that those 2^-28 below the largest keep their bits.  The largest itself, not what a norm allows: weights
// may be uneven, the norm's epsilon may rule, tables may scale.
constexpr float kUp = 8192.0f, kUpBits = 13.0f;
__device__ __forceinline__ float power_of(float most) { return power_below(fmaxf(most, 0x1p-113f)); }
// one over a power of two
__device__ __forceinline__ float inverse_power(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }

// head_rotation.cu: q_heads, then k_heads heads of `dim` from column 0 of proj on -> q, k [rows][heads][dim].  With q_factor (k_heads 0): q is fp16
// [rows][heads][ldq], zeros behind a head, each head divided by a power of two, q_factor [rows][heads], that leaves its numbers below 2^14.
struct RotationCall {
    const float* proj;
    int ld, q_heads, k_heads, dim;
    const int32_t *slots, *positions;
    int n_seq, n_tok;
    float eps;
    void *q, *k;
    float* q_factor;
    int ldq;
};
int launch_head_rotation(const tbl_head_rotation& r, int precision, const RotationCall& c, cudaStream_t st);

}  // namespace stack
}  // namespace tbl
