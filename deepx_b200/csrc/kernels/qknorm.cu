// dx_qknorm_rope: the norm of each head of the queries and keys and the rotation by their positions, in one pass.
//
//   y = w * x / sqrt(mean(x^2) + eps);   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin) for each pair (a, b) of the rotated part
//
// Bound by memory: every element is read once and written once.  The angles are one set for all heads of a token, so a block
// works them out once into shared memory: position * inv_freq is a float64 product (a float32 one is off by a tenth of a
// radian at a position of a million), reduced to a fraction of a turn there and turned into sine and cosine in float32.
//
// Measured (B200, inputs of other passes in between): 16384 tokens of 32 + 8 heads of 128, bf16: 62.9 us, 5.3 TB/s of the copy's 6.5.  A row's
// loads come while the row before is worked on (76 -> 71 us, with the short root), and two values are rounded with one instruction
// (71 -> 63 us): issue slots count here as much as bytes.  64 tokens: 3.6 us on the device, a launch's latency.
#include "common.cuh"

namespace dx {
namespace {

constexpr int CTA = 256;

struct RopeArgs {
    const void *q, *k, *qw, *kw;
    void *qo, *ko;
    int64_t q_stride, k_stride, qo_stride, ko_stride, tokens;
    int q_heads, k_heads, dim, rotated, interleaved, norm;
    float eps;
    const float *inv_freq;
    const void *positions;
    int pos64;
};

__device__ __forceinline__ double position(const RopeArgs &a, int64_t token) {
    return a.pos64 ? double(static_cast<const int64_t *>(a.positions)[token]) : double(static_cast<const int32_t *>(a.positions)[token]);
}
// (cosine, sine) of the angle pos * inv_freq
__device__ __forceinline__ float2 turn_of(double pos, float inv_freq) {
    const double turns = pos * double(inv_freq) * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * float(turns - rint(turns)), &s, &c);
    return make_float2(c, s);
}

// Any head size, stride and alignment: a warp takes a head, its elements in shared memory.
template <typename T> __global__ void __launch_bounds__(CTA) qknorm_rope_any_kernel(RopeArgs a) {
    __shared__ float2 cs[DX_ROPE_MAX_DIM / 2];
    __shared__ float row[CTA / 32][DX_ROPE_MAX_DIM];
    const int64_t token = blockIdx.x;
    griddep_wait_cta();
    for (int i = threadIdx.x; i < a.rotated / 2; i += CTA) cs[i] = turn_of(position(a, token), a.inv_freq[i]);
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *y = row[warp];
    for (int h = warp; h < a.q_heads + a.k_heads; h += CTA / 32) {
        const bool is_q = h < a.q_heads;
        const T *x = is_q ? static_cast<const T *>(a.q) + token * a.q_stride + int64_t(h) * a.dim
                          : static_cast<const T *>(a.k) + token * a.k_stride + int64_t(h - a.q_heads) * a.dim;
        T *o = is_q ? static_cast<T *>(a.qo) + token * a.qo_stride + int64_t(h) * a.dim
                    : static_cast<T *>(a.ko) + token * a.ko_stride + int64_t(h - a.q_heads) * a.dim;
        const T *w = static_cast<const T *>(is_q ? a.qw : a.kw);
        float sum = 0.f;
        for (int i = lane; i < a.dim; i += 32) {
            const float f = to_compute(x[i]);
            y[i] = f;
            sum += f * f;
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        const float r = a.norm ? 1.f / sqrtf(sum / float(a.dim) + a.eps) : 1.f;
        for (int i = lane; i < a.dim; i += 32) {
            float f = y[i] * r;
            if (a.norm && w) f *= to_compute(w[i]);
            y[i] = f;
        }
        __syncwarp();
        for (int i = lane; i < a.rotated / 2; i += 32) {
            const int p = a.interleaved ? 2 * i : i, q = a.interleaved ? 2 * i + 1 : i + a.rotated / 2;
            const float2 t = cs[i];
            const float u = y[p], v = y[q];
            o[p] = from_compute<T>(u * t.x - v * t.y);
            o[q] = from_compute<T>(v * t.x + u * t.y);
        }
        for (int i = a.rotated + lane; i < a.dim; i += 32) o[i] = from_compute<T>(y[i]);
        __syncwarp();
    }
}

// Whole 16-byte vectors: LANES threads share a head, each with one UNIT of sixteen elements, two chunks of eight.  In the rotated
// part a unit is a chunk and its partner half the rotated part further (or, interleaved, two chunks side by side): both elements of
// every pair are in one thread, so the rotation needs no exchange.  A block takes `per_block` tokens, whose angles are in shared
// memory; the first head's elements are loaded before the angles are worked out.
template <typename T> struct Eight {
    static constexpr int N = 16 / sizeof(T), P = 8 / N;
    Pack<T, N> p[P];
    __device__ __forceinline__ void load(const T *x) {
#pragma unroll
        for (int i = 0; i < P; ++i) p[i] = ld_stream<T, N>(x + i * N);
    }
    __device__ __forceinline__ void store(T *x) const {
#pragma unroll
        for (int i = 0; i < P; ++i) st_stream<T, N>(x + i * N, p[i]);
    }
    __device__ __forceinline__ float get(int e) const { return to_compute(p[e / N].v[e % N]); }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {  // two at a time: one conversion
            if constexpr (std::is_same<T, bf16>::value) *reinterpret_cast<__nv_bfloat162 *>(&p[e / N].v[e % N]) = __floats2bfloat162_rn(f[e], f[e + 1]);
            else if constexpr (std::is_same<T, f16>::value) *reinterpret_cast<__half2 *>(&p[e / N].v[e % N]) = __floats2half2_rn(f[e], f[e + 1]);
            else p[e / N].v[e % N] = f[e], p[(e + 1) / N].v[(e + 1) % N] = f[e + 1];
        }
    }
};

template <typename T, int LANES, bool INTERLEAVED> __global__ void __launch_bounds__(CTA) qknorm_rope_kernel(RopeArgs a, int per_block, FastDiv by_heads) {
    extern __shared__ __align__(16) float shared[];
    // What a lane reads together lies LANES apart in fours, so that the lanes of a team touch different banks: two weights [4][LANES], then
    // for each token [4][LANES] of two (cosine, sine).
    float4 *const weights = reinterpret_cast<float4 *>(shared), *const cs = weights + 2 * 4 * LANES;
    griddep_wait_cta();
    const int heads = a.q_heads + a.k_heads, half = a.rotated / 2;
    const int64_t token0 = int64_t(blockIdx.x) * per_block;
    const int tokens = int(min(int64_t(per_block), a.tokens - token0));
    const int team = threadIdx.x / LANES, u = threadIdx.x % LANES;
    const int chunks = a.dim / 8, rotated_units = INTERLEAVED ? 0 : half / 8;
    const bool apart = u < rotated_units;  // the rest: two chunks side by side
    const int first = apart ? u : 2 * u, second = apart ? u + rotated_units : 2 * u + 1;
    const bool has0 = first < chunks, has1 = second < chunks;
    const int rows = tokens * heads;
    const T *const q = static_cast<const T *>(a.q) + token0 * a.q_stride, *const k = static_cast<const T *>(a.k) + token0 * a.k_stride;
    T *const qo = static_cast<T *>(a.qo) + token0 * a.qo_stride, *const ko = static_cast<T *>(a.ko) + token0 * a.ko_stride;
    Eight<T> x0, x1;
    const float zeros[8] = {};
    x0.set(zeros);  // what a short last unit does not have stays zero
    x1.set(zeros);
    auto load = [&](int row) {
        const int t = int(fd_div(uint32_t(row), by_heads)), h = row - t * heads;
        const T *x = h < a.q_heads ? q + t * a.q_stride + h * a.dim : k + t * a.k_stride + (h - a.q_heads) * a.dim;
        if (has0) x0.load(x + first * 8);
        if (has1) x1.load(x + second * 8);
    };
    if (team < rows) load(team);
    if (a.norm) {
        for (int i = threadIdx.x; i < 2 * a.dim; i += CTA) {
            const bool is_k = i >= a.dim;
            const int d = i - (is_k ? a.dim : 0), chunk = d / 8;
            const T *w = static_cast<const T *>(is_k ? a.kw : a.qw);
            // of which unit's first or second chunk it is
            const bool split = chunk < 2 * rotated_units;
            const int unit = split && chunk >= rotated_units ? chunk - rotated_units : split ? chunk : chunk / 2, which = split ? chunk >= rotated_units : chunk & 1;
            reinterpret_cast<float *>(weights + ((is_k ? 4 : 0) + 2 * which + d % 8 / 4) * LANES + unit)[d % 4] = w ? to_compute(w[d]) : 1.f;
        }
    }
    for (int i = threadIdx.x; i < tokens * half; i += CTA) {
        const int t = i / half, f = i - t * half, unit = f / 8, e = f % 8;  // pair f: both orders have eight pairs of a unit in order
        reinterpret_cast<float2 *>(cs + (t * 4 + e / 2) * LANES + unit)[e & 1] = turn_of(position(a, token0 + t), a.inv_freq[f]);
    }
    __syncthreads();
    const float by_dim = 1.f / float(a.dim);
    // every thread of a warp takes the same number of turns: the sums are warp shuffles
    for (int row0 = 0; row0 < rows; row0 += CTA / LANES) {
        const int row = row0 + team;
        const bool live = row < rows;
        float y0[8], y1[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            y0[e] = x0.get(e);
            y1[e] = x1.get(e);
            sum += y0[e] * y0[e];
            sum += y1[e] * y1[e];
        }
        if (row + CTA / LANES < rows) load(row + CTA / LANES);  // the next row comes while this one is worked on
        const int t = int(fd_div(uint32_t(row), by_heads)), h = row - t * heads;
        const bool is_q = h < a.q_heads;
        if (a.norm) {
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            // 16-bit results do not show the 2^-22 that the short form is off by; the long one is two dozen instructions
            const float mean = sum * by_dim + a.eps, r = sizeof(T) == 4 ? 1.f / sqrtf(mean) : rsqrtf(mean);
            const float4 *w = weights + (is_q ? 0 : 4 * LANES) + u;
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 w0 = w[e / 4 * LANES], w1 = w[(2 + e / 4) * LANES];
                const float m0[4] = {w0.x, w0.y, w0.z, w0.w}, m1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    y0[e + d] *= r * m0[d];
                    y1[e + d] *= r * m1[d];
                }
            }
        }
        if (!live) continue;
        const float4 *turn = cs + t * 4 * LANES + u;
        if constexpr (INTERLEAVED) {
            auto rotate = [&](float (&y)[8], int chunk, int from) {
                if (chunk * 8 >= a.rotated) return;
#pragma unroll
                for (int p = 0; p < 4; p += 2) {
                    const float4 c = turn[(from + p / 2) * LANES];
                    const float s = y[2 * p], v = y[2 * p + 1], z = y[2 * p + 2], w = y[2 * p + 3];
                    y[2 * p] = s * c.x - v * c.y;
                    y[2 * p + 1] = v * c.x + s * c.y;
                    y[2 * p + 2] = z * c.z - w * c.w;
                    y[2 * p + 3] = w * c.z + z * c.w;
                }
            };
            rotate(y0, first, 0);
            rotate(y1, second, 2);
        } else if (apart) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float4 c = turn[e / 2 * LANES];
                const float s = y0[e], v = y1[e], z = y0[e + 1], w = y1[e + 1];
                y0[e] = s * c.x - v * c.y;
                y1[e] = v * c.x + s * c.y;
                y0[e + 1] = z * c.z - w * c.w;
                y1[e + 1] = w * c.z + z * c.w;
            }
        }
        T *o = is_q ? qo + t * a.qo_stride + h * a.dim : ko + t * a.ko_stride + (h - a.q_heads) * a.dim;
        Eight<T> z0, z1;
        z0.set(y0);
        z1.set(y1);
        if (has0) z0.store(o + first * 8);
        if (has1) z1.store(o + second * 8);
    }
}

template <typename T, int LANES> void launch_lanes(const RopeArgs &a, cudaStream_t st) {
    // enough blocks for every SM's eight, then up to sixteen tokens each
    int per_block = 1;
    while (per_block < (LANES > 16 ? 8 : 16) && a.tokens > int64_t(sm_count()) * 8 * per_block) per_block *= 2;
    const unsigned grid = unsigned((a.tokens + per_block - 1) / per_block);
    const size_t smem = size_t(2 + per_block) * 4 * LANES * sizeof(float4);
    const FastDiv by_heads = make_fastdiv(unsigned(a.q_heads + a.k_heads));
    if (a.interleaved) launch_pdl(qknorm_rope_kernel<T, LANES, true>, dim3(grid), dim3(CTA), smem, st, a, per_block, by_heads);
    else launch_pdl(qknorm_rope_kernel<T, LANES, false>, dim3(grid), dim3(CTA), smem, st, a, per_block, by_heads);
}

template <typename T> void launch_rope(const RopeArgs &a, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    bool vec = a.dim % 8 == 0 && a.rotated % (a.interleaved ? 8 : 16) == 0;
    for (const void *p : {a.q, a.k, a.qw, a.kw, static_cast<const void *>(a.qo), static_cast<const void *>(a.ko)}) vec = vec && aligned_to(p, 16);
    for (int64_t stride : {a.q_heads ? a.q_stride : 0, a.k_heads ? a.k_stride : 0, a.q_heads ? a.qo_stride : 0, a.k_heads ? a.ko_stride : 0}) vec = vec && stride % N == 0;
    if (!vec) {
        launch_pdl(qknorm_rope_any_kernel<T>, dim3(unsigned(a.tokens)), dim3(CTA), 0, st, a);
        return;
    }
    const int units = (a.dim + 15) / 16;
    if (units <= 4) launch_lanes<T, 4>(a, st);
    else if (units <= 8) launch_lanes<T, 8>(a, st);
    else if (units <= 16) launch_lanes<T, 16>(a, st);
    else launch_lanes<T, 32>(a, st);
}

}  // namespace
}  // namespace dx

extern "C" int dx_qknorm_rope(int dtype, const void *q, int64_t q_stride, int64_t q_heads, const void *k, int64_t k_stride, int64_t k_heads,
                              int64_t tokens, int64_t head_dim, int norm, const void *q_weight, const void *k_weight, double eps,
                              const float *inv_freq, int64_t rotated, int interleaved, int pos_dtype, const void *positions, void *q_out,
                              int64_t q_out_stride, void *k_out, int64_t k_out_stride, void *stream) {
    using namespace dx;
    if (dtype != DX_F32 && dtype != DX_F16 && dtype != DX_BF16) return fail(DX_E_DTYPE, "qknorm_rope: unsupported dtype code %d (float32, float16, bfloat16)", dtype);
    if (pos_dtype != DX_I32 && pos_dtype != DX_I64) return fail(DX_E_DTYPE, "qknorm_rope: positions must be int32 or int64");
    if (head_dim < 1 || head_dim > DX_ROPE_MAX_DIM) return fail(DX_E_SHAPE, "qknorm_rope: head_dim %lld (1 to %d)", (long long)head_dim, DX_ROPE_MAX_DIM);
    if (rotated < 0 || rotated > head_dim || rotated % 2) return fail(DX_E_SHAPE, "qknorm_rope: %lld rotated of %lld dimensions", (long long)rotated, (long long)head_dim);
    if (q_heads < 0 || k_heads < 0 || q_heads + k_heads > (1 << 20)) return fail(DX_E_SHAPE, "qknorm_rope: %lld and %lld heads", (long long)q_heads, (long long)k_heads);
    if (tokens < 0 || tokens > INT32_MAX) return fail(DX_E_SHAPE, "qknorm_rope: %lld tokens", (long long)tokens);
    if (norm && !(eps >= 0)) return fail(DX_E_ARG, "qknorm_rope: eps %g", eps);
    if (tokens == 0 || q_heads + k_heads == 0) return DX_OK;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || (rotated && (!inv_freq || !positions))) return fail(DX_E_ARG, "qknorm_rope: null tensor pointer");
    const int64_t es = dx_dtype_size(dtype);
    struct Side {
        const void *in;
        void *out;
        int64_t stride, out_stride, heads;
    } sides[2] = {{q, q_out, q_stride, q_out_stride, q_heads}, {k, k_out, k_stride, k_out_stride, k_heads}};
    for (const Side &x : sides)
        if (x.heads && (x.stride < x.heads * head_dim || x.out_stride < x.heads * head_dim)) return fail(DX_E_SHAPE, "qknorm_rope: rows overlap at strides %lld and %lld", (long long)x.stride, (long long)x.out_stride);
    // An output may be its own input, or stand beside other tensors' columns in the rows of one buffer (a packed projection); it meets nothing else.
    const int64_t wide = head_dim * es;
    const Span others[] = {span(norm ? q_weight : nullptr, wide), span(norm ? k_weight : nullptr, wide), span(rotated ? inv_freq : nullptr, rotated / 2 * 4),
                           span(rotated ? positions : nullptr, tokens * dx_dtype_size(pos_dtype))};
    auto out_of = [&](const Side &x) { return span(x.heads ? x.out : nullptr, tokens, x.out_stride * es, x.heads * wide); };
    if (meet(out_of(sides[0]), out_of(sides[1]))) return fail(DX_E_ALIAS, "qknorm_rope: the outputs overlap");
    for (const Side &o : sides) {
        for (const Side &i : sides) {
            const bool own = &o == &i && o.out == i.in && o.out_stride == i.stride;
            if (!own && meet(out_of(o), span(i.heads ? i.in : nullptr, tokens, i.stride * es, i.heads * wide)))
                return fail(DX_E_ALIAS, "qknorm_rope: an output overlaps an input other than its own");
        }
        for (const Span &x : others)
            if (meet(out_of(o), x)) return fail(DX_E_ALIAS, "qknorm_rope: an output overlaps a weight, inv_freq or positions");
    }
    RopeArgs a{q, k, q_weight, k_weight, q_out, k_out, q_stride, k_stride, q_out_stride, k_out_stride, tokens, int(q_heads), int(k_heads),
               int(head_dim), int(rotated), interleaved, norm, float(eps), inv_freq, positions, pos_dtype == DX_I64};
    cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case DX_F32: launch_rope<float>(a, st); break;
        case DX_F16: launch_rope<f16>(a, st); break;
        default: launch_rope<bf16>(a, st); break;
    }
    return check_launch("qknorm_rope");
}
