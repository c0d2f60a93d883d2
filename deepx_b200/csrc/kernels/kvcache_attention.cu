// dx_kvcache_attention: attention of packed new tokens over an 8-bit paged cache.
//
//   out[t,h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q[t,h].k_j - m),   m the running maximum,   j <= pos(t), j > pos(t) - window
#include "kvcache.cuh"

namespace dx {
namespace kv {
namespace {

constexpr int CTA = 128;

struct Attn {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    int q_heads, group, window;
    float scale;
    int32_t *flag;
};

// A warp takes one head of one row and walks its keys.
template <typename T, int FMT> __global__ void __launch_bounds__(CTA) attention_row_kernel(Attn a, Cache c, Seqs s) {
    if (blockIdx.x == 0) check_seqs(s, c, a.flag);
    const int lane = threadIdx.x & 31;
    const int64_t unit = int64_t(blockIdx.x) * (CTA / 32) + (threadIdx.x >> 5);
    if (unit >= s.rows * a.q_heads) return;
    const int64_t row = unit / a.q_heads;
    const int h = int(unit - row * a.q_heads), kh = h / a.group;
    const int b = seq_of_row(s.starts, s.batch, row);
    if (b < 0) return;
    const Seq sq = seq_at(s, c, b);
    const int64_t i = row - sq.row0;
    if (i < 0 || i >= sq.n) return;
    const int64_t pos = sq.first + i;
    const T *q = static_cast<const T *>(a.q) + row * a.q_stride + int64_t(h) * c.dim;
    const int units = c.dim / 4;  // lane: four dimensions at 4 * lane, four at 128 + 4 * lane
    float qv[8], o[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int d = (j / 4) * 128 + lane * 4 + j % 4;
        qv[j] = d < c.dim ? to_compute(q[d]) : 0.f;
    }
    float m = -__int_as_float(0x7f800000), l = 0.f;
    const int end = int(min(int64_t(sq.end), pos + 1));
    const int begin = a.window > 0 ? int(max(int64_t(0), pos - a.window + 1)) : 0;
    int64_t page = -1;
    for (int j = begin; j < end; ++j) {
        if (j == begin || (j & (c.page - 1)) == 0) page = page_at(s, c, b, j, a.flag);
        if (page < 0) continue;
        const int64_t at = ((page * c.heads + kh) * c.page + (j & (c.page - 1))) * c.dim;
        float kf[8], vf[8];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const bool in = p * 32 + lane < units;
            const uint32_t kw = in ? *reinterpret_cast<const uint32_t *>(c.k + at + p * 128 + lane * 4) : 0u;
            const uint32_t vw = in ? *reinterpret_cast<const uint32_t *>(c.v + at + p * 128 + lane * 4) : 0u;
            const float2 k0 = __half22float2(decode2<FMT>(kw & 0xFFFFu)), k1 = __half22float2(decode2<FMT>(kw >> 16));
            const float2 v0 = __half22float2(decode2<FMT>(vw & 0xFFFFu)), v1 = __half22float2(decode2<FMT>(vw >> 16));
            kf[4 * p] = k0.x, kf[4 * p + 1] = k0.y, kf[4 * p + 2] = k1.x, kf[4 * p + 3] = k1.y;
            vf[4 * p] = v0.x, vf[4 * p + 1] = v0.y, vf[4 * p + 2] = v1.x, vf[4 * p + 3] = v1.y;
        }
        float dot = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) dot += qv[d] * kf[d];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        const float x = dot * c.k_scale[page * c.heads + kh] * a.scale;
        const float top = fmaxf(m, x);
        const float turn = m == top ? 1.f : __expf(m - top), p = __expf(x - top);
        const float w = p * c.v_scale[page * c.heads + kh];
        m = top;
        l = l * turn + p;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] = o[d] * turn + w * vf[d];
    }
    T *out = static_cast<T *>(a.out) + row * a.out_stride + int64_t(h) * c.dim;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int d = (j / 4) * 128 + lane * 4 + j % 4;
        if (d < c.dim) out[d] = from_compute<T>(l == 0.f ? 0.f : o[j] / l);
    }
}

}  // namespace
}  // namespace kv
}  // namespace dx

extern "C" size_t dx_kvcache_attention_workspace_bytes(int dtype, int64_t q_heads, const dx_kvseqs *seqs, const dx_kvcache *cache, int64_t max_new) {
    return 0;
}

extern "C" int dx_kvcache_attention(int dtype, const void *q, int64_t q_stride, int64_t q_heads, const dx_kvseqs *seqs, const dx_kvcache *cache,
                                    double scale, int64_t max_new, int64_t window, void *out, int64_t out_stride, void *workspace,
                                    size_t workspace_bytes, int32_t *flag, void *stream) {
    using namespace dx;
    kv::Cache c;
    kv::Seqs s;
    if (int e = kv::check("kvcache_attention", cache, seqs, &c, &s)) return e;
    if (dtype != DX_F16 && dtype != DX_BF16) return fail(DX_E_DTYPE, "kvcache_attention: unsupported dtype code %d (float16, bfloat16)", dtype);
    if (q_heads < 1 || q_heads % c.heads || q_heads > 65535) return fail(DX_E_SHAPE, "kvcache_attention: %lld query heads over %d key heads", (long long)q_heads, c.heads);
    const int64_t width = q_heads * c.dim;
    if (q_stride < width || out_stride < width) return fail(DX_E_SHAPE, "kvcache_attention: rows of %lld elements overlap at strides %lld and %lld", (long long)width, (long long)q_stride, (long long)out_stride);
    if (!(scale > 0) || !(float(scale) > 0) || scale > 3e38) return fail(DX_E_ARG, "kvcache_attention: scale %g", scale);
    if (max_new < 0 || window < 0) return fail(DX_E_ARG, "kvcache_attention: max_new %lld, window %lld", (long long)max_new, (long long)window);
    if (s.rows == 0 || s.batch == 0) return DX_OK;
    if (!q || !out) return fail(DX_E_ARG, "kvcache_attention: null tensor pointer");
    const int64_t qb = ((s.rows - 1) * q_stride + width) * 2, ob = ((s.rows - 1) * out_stride + width) * 2;
    const int64_t codes = c.pages * c.heads * int64_t(c.page) * c.dim;
    if (kv::overlap(q, qb, out, ob) || kv::overlap(out, ob, c.k, codes) || kv::overlap(out, ob, c.v, codes))
        return fail(DX_E_ALIAS, "kvcache_attention: the output overlaps an input");
    kv::Attn a{q, out, q_stride, out_stride, int(q_heads), int(q_heads / c.heads), int(window > INT32_MAX ? 0 : window), float(scale), flag};
    cudaStream_t st = as_stream(stream);
    const unsigned grid = unsigned((s.rows * q_heads + 3) / 4);
    if (dtype == DX_F16) {
        if (cache->format == DX_CACHE_I8) kv::attention_row_kernel<f16, DX_CACHE_I8><<<grid, kv::CTA, 0, st>>>(a, c, s);
        else kv::attention_row_kernel<f16, DX_CACHE_E4M3><<<grid, kv::CTA, 0, st>>>(a, c, s);
    } else {
        if (cache->format == DX_CACHE_I8) kv::attention_row_kernel<bf16, DX_CACHE_I8><<<grid, kv::CTA, 0, st>>>(a, c, s);
        else kv::attention_row_kernel<bf16, DX_CACHE_E4M3><<<grid, kv::CTA, 0, st>>>(a, c, s);
    }
    return check_launch("kvcache_attention");
}
