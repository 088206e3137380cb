// Attention over a 4-bit cache in fp32 arithmetic: any head size, any number of query rows.
//
// A CTA has up to 16 query rows that share a key/value head and a split of the context; each of its four warps takes tiles of 32 tokens by itself,
// with its own maxima, sums and outputs.  For the scores a lane has a token and turns its codes into numbers sixteen at a time (one scale), for all
// rows at once; for the outputs a lane has neighbouring dimensions, and the tokens' weights come from shared memory.  Cached numbers so are read as
// they lie, 4 bits each, once per 16 rows.  Bound by latency: eight warps to an SM at sixteen rows (254 registers) leave 56 % of the issue slots and
// 71 % of the multiplications' pipe unused while rows come (200 tokens behind 500, 32 and 8 heads of 128: 182 us), and few tokens take the chain of one
// tile a warp (five sequences of three tokens over 777: 27 us, this kernel 15).
#include "quantized.cuh"

namespace tbl {
namespace stack {
namespace {

constexpr int kWarps = 4, kTile = 32, kThreads = 32 * kWarps;

// W: the head size rounded up to 64, in sixty-fours; R: query rows
template <typename T, int W, int R>
__global__ void __launch_bounds__(kThreads) quantized_rows_kernel(const QuantizedParams p) {
    constexpr int DP = 64 * W, kDims = 2 * W;                    // dimensions of a lane's share of an output
    __shared__ __align__(16) float room[kWarps * R * DP];        // queries and weights, then the outputs
    float(*q_s)[DP] = reinterpret_cast<float(*)[DP]>(room);
    float(*w_s)[R][kTile] = reinterpret_cast<float(*)[R][kTile]>(room + R * DP);
    float(*o_s)[R][DP] = reinterpret_cast<float(*)[R][DP]>(room);
    static_assert(R * DP + kWarps * R * kTile <= kWarps * R * DP, "queries and weights have room");
    __shared__ float m_s[kWarps][R], l_s[kWarps][R];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int seq = blockIdx.x / p.G, g = blockIdx.x % p.G, first = blockIdx.y * R, split = blockIdx.z, total = p.n_tok * p.group;
    pdl_wait();
    const int slot = p.slots[seq], pos0 = p.positions[slot];
    const int n = min(pos0 + min(total - 1, first + R - 1) / p.group + 1, p.capacity);           // tokens the last row sees
    const int per = ((n + p.splits - 1) / p.splits + kTile - 1) / kTile * kTile;
    const int t0 = min(split * per, max(n, 0)), t1 = min(n, t0 + per);
    const float* queries = static_cast<const float*>(p.q);
    for (int i = tid; i < R * DP; i += kThreads) {
        const int r = i / DP, c = i % DP, at = first + r;
        q_s[r][c] = at < total && c < p.d ? queries[((static_cast<size_t>(seq) * p.n_tok + at / p.group) * p.H + g * p.group + at % p.group) * p.ldq + c] : 0.0f;
    }
    __syncthreads();
    const uint8_t* cache = quantized_at(p, slot, g, 0);
    float m[R], l[R], o[R][kDims];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int e = 0; e < kDims; ++e) o[r][e] = 0.0f;
    }
    for (int t = t0 + warp * kTile; t < t1; t += kThreads) {
        const int token = t + lane;
        const uint8_t* row = cache + static_cast<size_t>(min(token, t1 - 1)) * p.row;
        float s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = 0.0f;
#pragma unroll 2
        for (int c = 0; c < DP / 16; ++c) {
            const uint2 codes = *reinterpret_cast<const uint2*>(row + 8 * c);
            const float scale = scale_of(row[DP + c]);
            float k[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 f = __half22float2(codes_of(((i < 4 ? codes.x : codes.y) >> (8 * (i & 3))) & 0xffu));
                k[2 * i] = f.x * scale;
                k[2 * i + 1] = f.y * scale;
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 q = *reinterpret_cast<const float4*>(&q_s[r][16 * c + i]);
                    s[r] = fmaf(q.x, k[i], s[r]); s[r] = fmaf(q.y, k[i + 1], s[r]); s[r] = fmaf(q.z, k[i + 2], s[r]); s[r] = fmaf(q.w, k[i + 3], s[r]);
                }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int last = min(pos0 + min(first + r, total - 1) / p.group, t1 - 1);
            const float x = token <= last ? s[r] * p.scale_log2 : -INFINITY, mn = fmaxf(m[r], warp_max(x));
            // a row that has seen nothing yet keeps its maximum at -infinity and its weights at zero (a score that is NaN has no maximum, but its weight)
            const float f = m[r] == -INFINITY ? 0.0f : exp2f(m[r] - mn), w = x == -INFINITY ? 0.0f : exp2f(x - mn);
            m[r] = mn;
            l[r] = fmaf(l[r], f, w);
            w_s[warp][r][lane] = w;
#pragma unroll
            for (int e = 0; e < kDims; ++e) o[r][e] *= f;
        }
        __syncwarp();
        // (tokens behind the split's end are not looked at: a weight of zero would need a finite value beside it)
        const int here = min(kTile, t1 - t);
        const uint8_t* values = cache + static_cast<size_t>(t) * p.row + DP / 2 + lane;           // numbers 2 lane, 2 lane + 1 of every 64
        const uint8_t* scales = cache + static_cast<size_t>(t) * p.row + DP + DP / 16 + lane / 8;
#pragma unroll 4
        for (int i = 0; i < here; ++i) {
            float v[kDims];
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float scale = scale_of(scales[static_cast<size_t>(i) * p.row + 4 * e]);
                const float2 f = __half22float2(codes_of(values[static_cast<size_t>(i) * p.row + 32 * e]));
                v[2 * e] = f.x * scale;
                v[2 * e + 1] = f.y * scale;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float w = w_s[warp][r][i];
#pragma unroll
                for (int e = 0; e < kDims; ++e) o[r][e] = fmaf(w, v[e], o[r][e]);
            }
        }
        __syncwarp();
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = warp_sum(l[r]);
        if (lane == 0) { m_s[warp][r] = m[r]; l_s[warp][r] = sum; }
#pragma unroll
        for (int e = 0; e < W; ++e) *reinterpret_cast<float2*>(&o_s[warp][r][64 * e + 2 * lane]) = make_float2(o[r][2 * e], o[r][2 * e + 1]);
    }
    __syncthreads();
    const int rows = min(R, total - first);
    for (int i = tid; i < rows * p.d; i += kThreads) {
        const int r = i / p.d, c = i - r * p.d, at = first + r, head = g * p.group + at % p.group;
        const size_t row = static_cast<size_t>(seq) * p.n_tok + at / p.group;
        float top = m_s[0][r], v = 0.0f, sum = 0.0f;
#pragma unroll
        for (int k = 1; k < kWarps; ++k) top = fmaxf(top, m_s[k][r]);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            const float w = m_s[k][r] == -INFINITY ? 0.0f : exp2f(m_s[k][r] - top);
            v = fmaf(o_s[k][r][c], w, v);
            sum = fmaf(l_s[k][r], w, sum);
        }
        if (p.splits > 1) {
            const size_t u = (row * p.H + head) * p.splits + split;
            if (c == 0) { p.part_m[u] = top; p.part_l[u] = sum; }
            p.part_o[u * p.ldo + c] = v;
        } else {
            const float gate = p.g_off < 0 ? 1.0f : sigmoid_f(p.proj[row * p.ld + p.g_off + head * p.d + c]);
            static_cast<T*>(p.out)[(row * p.H + head) * p.d + c] = from_f<T>(v * (p.value_unit / sum) * gate);
        }
    }
}

// Query rows of a CTA.  Many of them share what a cached number costs; few of them are done sooner, where the CTAs at hand (`tiles`: splits at most,
// times sequences and key/value heads) leave SMs empty (fp32, sixteen rows and as here: five sequences of three tokens over 777, 10 and 2 heads of
// 90, 28 and 22 us; four tokens over 300, 32 and 8 heads of 128, 27 and 17; 16 over 4000, 8 and 2 heads, 34 with sixteen rows, 36 with eight).
int rows_of(int width, long long total, long long tiles) {
    int r = total <= 4 ? 4 : total <= 8 || width > 128 ? 8 : 16;
    while (r > 4 && tiles * ceil_div(total, r) < 3 * kNumSm / 2) r /= 2;
    return r;
}
long long tiles_of(int n_seq, int kv_heads, int context) { return static_cast<long long>(n_seq) * kv_heads * ceil_div(context, kWarps * kTile); }

template <typename T, int W, int R>
cudaError_t launch(const QuantizedParams& p, int n_seq, cudaStream_t st) {
    const dim3 grid(n_seq * p.G, ceil_div(static_cast<long long>(p.n_tok) * p.group, R), p.splits);
    if (grid.y > 65535 || grid.z > 65535) return cudaErrorInvalidValue;
    return launch_dependent(quantized_rows_kernel<T, W, R>, grid, dim3(kThreads), 0, st, p);
}
template <typename T, int W>
cudaError_t launch_rows(const QuantizedParams& p, int n_seq, cudaStream_t st) {
    const int r = rows_of(p.width, static_cast<long long>(p.n_tok) * p.group, tiles_of(n_seq, p.G, p.ctx));
    if constexpr (W <= 2) {
        if (r == 16) return launch<T, W, 16>(p, n_seq, st);
    }
    return r == 4 ? launch<T, W, 4>(p, n_seq, st) : launch<T, W, 8>(p, n_seq, st);
}
template <typename T>
cudaError_t launch_width(const QuantizedParams& p, int n_seq, cudaStream_t st) {
    switch (p.width) {
        case 64: return launch_rows<T, 1>(p, n_seq, st);
        case 128: return launch_rows<T, 2>(p, n_seq, st);
        case 192: return launch_rows<T, 3>(p, n_seq, st);
        default: return launch_rows<T, 4>(p, n_seq, st);
    }
}

}  // namespace

long long quantized_rows_blocks(const tbl_quantized_mixer& m, int n_seq, int n_tok, int context) {
    const long long total = static_cast<long long>(n_tok) * (m.heads / m.kv_heads);
    const int rows = rows_of(quantized_width(m.dim), total, tiles_of(n_seq, m.kv_heads, context));
    return (total + rows - 1) / rows;
}
int quantized_rows_splits(const tbl_quantized_mixer& m, int n_seq, int n_tok, int context) {
    const long long units = static_cast<long long>(n_seq) * m.kv_heads * quantized_rows_blocks(m, n_seq, n_tok, context);
    const int tokens = ceil_div(context, kWarps * kTile);        // a split is worth at least a tile of each warp
    long long s = 4LL * kNumSm / units;
    if (s > tokens) s = tokens;
    return s < 1 ? 1 : static_cast<int>(s < 1024 ? s : 1024);
}

int launch_quantized_rows(const QuantizedParams& p, int precision, int n_seq, cudaStream_t st) {
    return (precision == TBL_BF16 ? launch_width<bf16>(p, n_seq, st) : launch_width<float>(p, n_seq, st)) == cudaSuccess ? TBL_OK : TBL_ERR_CUDA;
}

}  // namespace stack
}  // namespace tbl
