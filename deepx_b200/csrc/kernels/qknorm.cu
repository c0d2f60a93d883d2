// dx_qknorm_rope: the norm of each head of the queries and keys and the rotation by their positions, in one pass.
//
//   y = w * x / sqrt(mean(x^2) + eps);   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin) for each pair (a, b) of the rotated part
//
// Bound by memory: every element is read once and written once.  The angles are one set for all heads of a token, so a block
// works them out once into shared memory: position * inv_freq is a float64 product (a float32 one is off by a tenth of a
// radian at a position of a million), reduced to a fraction of a turn there and turned into sine and cosine in float32.
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

__device__ __forceinline__ void angles(const RopeArgs &a, int64_t token, float2 *cs) {
    const double pos = a.pos64 ? double(static_cast<const int64_t *>(a.positions)[token]) : double(static_cast<const int32_t *>(a.positions)[token]);
    for (int i = threadIdx.x; i < a.rotated / 2; i += blockDim.x) {
        const double turns = pos * double(a.inv_freq[i]) * 0.15915494309189533577;  // 1 / (2 pi)
        float s, c;
        sincospif(2.f * float(turns - rint(turns)), &s, &c);
        cs[i] = make_float2(c, s);
    }
}

// Any head size, stride and alignment: a warp takes a head, its elements in shared memory.
template <typename T> __global__ void __launch_bounds__(CTA) qknorm_rope_any_kernel(RopeArgs a) {
    __shared__ float2 cs[DX_ROPE_MAX_DIM / 2];
    __shared__ float row[CTA / 32][DX_ROPE_MAX_DIM];
    const int64_t token = blockIdx.x;
    angles(a, token, cs);
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
    // A token's rows in one buffer (a packed projection) interleave with the other tensor's: only equal-stride rows that
    // do not share columns, or the very same rows, may.
    for (const Side &o : sides)
        for (const Side &i : sides) {
            if (!o.heads || !i.heads) continue;
            const bool same = &o == &i && o.out == i.in && o.out_stride == i.stride;
            const int64_t ow = o.heads * head_dim * es, iw = i.heads * head_dim * es;
            const char *a = static_cast<const char *>(o.out), *b = static_cast<const char *>(i.in);
            const int64_t ob = (tokens - 1) * o.out_stride * es + ow, ib = (tokens - 1) * i.stride * es + iw;
            if (same || a + ob <= b || b + ib <= a) continue;
            const int64_t pitch = o.out_stride * es;
            const int64_t shift = ((a - b) % pitch + pitch) % pitch;
            const bool apart = o.out_stride == i.stride && shift >= iw && shift + ow <= pitch;
            if (!apart) return fail(DX_E_ALIAS, "qknorm_rope: an output overlaps an input other than its own");
        }
    RopeArgs a{q, k, q_weight, k_weight, q_out, k_out, q_stride, k_stride, q_out_stride, k_out_stride, tokens, int(q_heads), int(k_heads),
               int(head_dim), int(rotated), interleaved, norm, float(eps), inv_freq, positions, pos_dtype == DX_I64};
    cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case DX_F32: qknorm_rope_any_kernel<float><<<unsigned(tokens), CTA, 0, st>>>(a); break;
        case DX_F16: qknorm_rope_any_kernel<f16><<<unsigned(tokens), CTA, 0, st>>>(a); break;
        default: qknorm_rope_any_kernel<bf16><<<unsigned(tokens), CTA, 0, st>>>(a); break;
    }
    return check_launch("qknorm_rope");
}
