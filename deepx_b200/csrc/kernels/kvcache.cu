// dx_kvcache_write and dx_kvcache_read: values into the pages of an 8-bit key/value cache, and back.
//
// Both are bound by memory: a value is read (written) once at its type's size, its code written (read) once.
#include "kvcache.cuh"

namespace dx {
namespace kv {

int check(const char *what, const dx_kvcache *c, const dx_kvseqs *s, Cache *cache, Seqs *seqs) {
    if (!c || !s) return fail(DX_E_ARG, "%s: null descriptor", what);
    if (c->format < 0 || c->format >= DX_CACHE_FORMAT_COUNT) return fail(DX_E_DTYPE, "%s: unknown cache format %d", what, c->format);
    const int64_t p = c->page_tokens;
    if (p < 16 || p > 256 || (p & (p - 1))) return fail(DX_E_SHAPE, "%s: pages of %lld tokens (16, 32, 64, 128 or 256)", what, (long long)p);
    if (c->head_dim < 16 || c->head_dim > MAX_DIM || c->head_dim % 16)
        return fail(DX_E_SHAPE, "%s: head_dim %lld is no multiple of 16 up to %d", what, (long long)c->head_dim, MAX_DIM);
    if (c->kv_heads < 1 || c->kv_heads > 65535) return fail(DX_E_SHAPE, "%s: %lld key heads", what, (long long)c->kv_heads);
    if (c->pages < 0 || c->pages > INT32_MAX) return fail(DX_E_SHAPE, "%s: %lld pages", what, (long long)c->pages);
    if (s->batch < 0 || s->batch > (1 << 24) || s->rows < 0 || s->rows > INT32_MAX || s->table_cols < 0 || s->table_cols > INT32_MAX / p)
        return fail(DX_E_SHAPE, "%s: batch %lld, rows %lld, table of %lld columns", what, (long long)s->batch, (long long)s->rows, (long long)s->table_cols);
    if (s->batch > 0 && s->rows > 0) {
        if (!s->starts || !s->lens || (!s->table && s->table_cols > 0)) return fail(DX_E_ARG, "%s: null starts, lens or table", what);
        if (c->pages > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return fail(DX_E_ARG, "%s: null cache pointer", what);
        if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16)) return fail(DX_E_ARG, "%s: the cache must start on a 16-byte boundary", what);
    }
    *cache = Cache{static_cast<uint8_t *>(c->k), static_cast<uint8_t *>(c->v), c->k_scale, c->v_scale, c->pages, int(c->kv_heads), int(p),
                   __builtin_ctzll(uint64_t(p)), int(c->head_dim)};
    *seqs = Seqs{s->starts, s->lens, s->table, int(s->batch), int(s->table_cols), s->rows};
    return DX_OK;
}

namespace {

constexpr int W_CTA = 128;
constexpr int MAX_CHUNK = 128;

template <typename T> __device__ __forceinline__ float4 load4(const T *p, bool vec) {
    if (vec) {
        const Pack<T, 4> v = ld_cached<T, 4>(p);
        return make_float4(to_compute(v.v[0]), to_compute(v.v[1]), to_compute(v.v[2]), to_compute(v.v[3]));
    }
    return make_float4(to_compute(p[0]), to_compute(p[1]), to_compute(p[2]), to_compute(p[3]));
}

// A block takes the pages whose first new token is one of `chunk` packed rows, for one head, of the keys (blockIdx.z = 0) or
// the values: the largest size of the page's new values, the page's scale from it, the codes in a second pass over the
// same rows (which the first has left in L1 / L2).
template <typename T, int FMT>
__global__ void __launch_bounds__(W_CTA) write_kernel(const T *k, int64_t k_stride, const T *v, int64_t v_stride, Cache c, Seqs s, int chunk,
                                                      bool vec, int32_t *flag) {
    __shared__ int list[MAX_CHUNK], count;
    __shared__ float part[W_CTA / 32];
    const int head = blockIdx.y;
    const T *x = blockIdx.z ? v : k;
    const int64_t stride = blockIdx.z ? v_stride : k_stride;
    uint8_t *codes = blockIdx.z ? c.v : c.k;
    float *scales = blockIdx.z ? c.v_scale : c.k_scale;
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_seqs(s, c, flag);
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const int64_t row0 = int64_t(blockIdx.x) * chunk;
    if (int(threadIdx.x) < chunk && row0 + threadIdx.x < s.rows) {
        const int64_t row = row0 + threadIdx.x;
        const int b = seq_of_row(s.starts, s.batch, row);
        if (b >= 0) {
            const Seq q = seq_at(s, c, b);
            const int64_t i = row - q.row0;
            const int64_t pos = q.first + i;
            if (i >= 0 && i < q.n && pos >= 0 && pos < q.end && (i == 0 || pos == 0 || (pos & (c.page - 1)) == 0)) list[atomicAdd(&count, 1)] = int(row);
        }
    }
    __syncthreads();
    const int units = c.dim / 4;
    const int found = count;
    for (int n = 0; n < found; ++n) {
        const int64_t row = list[n];
        const int b = seq_of_row(s.starts, s.batch, row);
        const Seq q = seq_at(s, c, b);
        const int pos = int(q.first + (row - q.row0));
        const int slot = pos & (c.page - 1);
        const int tokens = int(min(int64_t(min(c.page - slot, q.end - pos)), q.n - (row - q.row0)));
        const int64_t page = page_at(s, c, b, pos, flag);
        if (page < 0) continue;  // the same answer in every thread
        const T *src = x + row * stride + int64_t(head) * c.dim;
        uint8_t *dst = codes + ((page * c.heads + head) * c.page) * int64_t(c.dim);
        float amax = 0.f;
        bool nan = false;
        for (int u = threadIdx.x; u < tokens * units; u += W_CTA) {
            const int t = u / units;
            const float4 a = load4(src + t * stride + (u - t * units) * 4, vec);
            auto size = [&](float f) {
                nan |= f != f;
                f = fabsf(f);
                return f < __int_as_float(0x7f800000) ? f : 0.f;
            };
            amax = fmaxf(amax, fmaxf(fmaxf(size(a.x), size(a.y)), fmaxf(size(a.z), size(a.w))));
        }
        if (nan) raise(flag, FLAG_NAN);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
        const float had = slot ? scales[page * c.heads + head] : 0.f;
        __syncthreads();  // every thread has read the old scale
#pragma unroll
        for (int w = 0; w < W_CTA / 32; ++w) amax = fmaxf(amax, part[w]);
        float scale = scale_for<FMT>(amax);
        if (slot) scale = fmaxf(scale, scale_kept(had));
        const float inv = inverse_of(scale);
        if (slot && scale != had) {  // the earlier tokens' codes in units of the grown scale
            const float by = had * inv;
            for (int u = threadIdx.x; u < slot * units; u += W_CTA) {
                uint32_t w = *reinterpret_cast<const uint32_t *>(dst + int64_t(u) * 4);
                const float2 lo = __half22float2(decode2<FMT>(w & 0xFFFFu)), hi = __half22float2(decode2<FMT>(w >> 16));
                w = encode4<FMT>(lo.x * by, lo.y * by, hi.x * by, hi.y * by);
                *reinterpret_cast<uint32_t *>(dst + int64_t(u) * 4) = w;
            }
        }
        for (int u = threadIdx.x; u < tokens * units; u += W_CTA) {
            const int t = u / units;
            const float4 a = load4(src + t * stride + (u - t * units) * 4, vec);
            *reinterpret_cast<uint32_t *>(dst + (int64_t(slot) * units + u) * 4) = encode4<FMT>(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        }
        if (threadIdx.x == 0) scales[page * c.heads + head] = scale;
        __syncthreads();  // `part` is free again
    }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(W_CTA) read_kernel(Cache c, Seqs s, T *k, int64_t k_stride, T *v, int64_t v_stride, bool vec, int32_t *flag) {
    if (blockIdx.x == 0 && blockIdx.y == 0) check_seqs(s, c, flag);
    const int64_t row = blockIdx.x;
    const int b = seq_of_row(s.starts, s.batch, row);
    if (b < 0) return;
    const Seq q = seq_at(s, c, b);
    const int64_t i = row - q.row0;
    if (i < 0 || i >= q.n) return;
    const int64_t pos = q.first + i;
    const int64_t page = pos >= 0 && pos < q.end ? page_at(s, c, b, int(pos), flag) : -1;
    const uint8_t *codes = blockIdx.y ? c.v : c.k;
    const float *scales = blockIdx.y ? c.v_scale : c.k_scale;
    T *out = blockIdx.y ? v + row * v_stride : k + row * k_stride;
    const int units = c.dim / 4;
    for (int u = threadIdx.x; u < c.heads * units; u += W_CTA) {
        const int h = u / units;
        Pack<T, 4> o;
        if (page < 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o.v[j] = from_compute<T>(0.f);
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + ((page * c.heads + h) * c.page + (pos & (c.page - 1))) * c.dim + (u - h * units) * 4);
            const float f = scales[page * c.heads + h];
            const float2 lo = __half22float2(decode2<FMT>(w & 0xFFFFu)), hi = __half22float2(decode2<FMT>(w >> 16));
            o.v[0] = from_compute<T>(lo.x * f);
            o.v[1] = from_compute<T>(lo.y * f);
            o.v[2] = from_compute<T>(hi.x * f);
            o.v[3] = from_compute<T>(hi.y * f);
        }
        T *dst = out + int64_t(u) * 4;
        if (vec) st_stream<T, 4>(dst, o);
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[j] = o.v[j];
        }
    }
}

int check_rows(const char *what, int dtype, const Seqs &s, const Cache &c, const void *k, int64_t k_stride, const void *v, int64_t v_stride) {
    if (dtype != DX_F32 && dtype != DX_F16 && dtype != DX_BF16) return fail(DX_E_DTYPE, "%s: unsupported dtype code %d (float32, float16, bfloat16)", what, dtype);
    const int64_t width = int64_t(c.heads) * c.dim;
    if (k_stride < width || v_stride < width) return fail(DX_E_SHAPE, "%s: rows of %lld elements overlap at strides %lld and %lld", what, (long long)width, (long long)k_stride, (long long)v_stride);
    if (s.rows == 0 || s.batch == 0) return DX_OK;
    if (!k || !v) return fail(DX_E_ARG, "%s: null tensor pointer", what);
    const int64_t es = dx_dtype_size(dtype), codes = c.pages * c.heads * int64_t(c.page) * c.dim;
    for (const void *p : {k, v}) {
        const int64_t bytes = ((s.rows - 1) * (p == k ? k_stride : v_stride) + width) * es;
        if (overlap(p, bytes, c.k, codes) || overlap(p, bytes, c.v, codes)) return fail(DX_E_ALIAS, "%s: a tensor overlaps the cache", what);
    }
    return DX_OK;
}

template <typename T> bool packs_of_4(const void *k, int64_t k_stride, const void *v, int64_t v_stride) {
    return k_stride % 4 == 0 && v_stride % 4 == 0 && aligned_to(k, 4 * sizeof(T)) && aligned_to(v, 4 * sizeof(T));
}

template <typename T, int FMT>
void launch_write(const void *k, int64_t ks, const void *v, int64_t vs, const Cache &c, const Seqs &s, int32_t *flag, cudaStream_t st) {
    int chunk = 1;
    while (chunk < MAX_CHUNK && chunk < c.page && int64_t(chunk) * s.batch < s.rows) chunk *= 2;
    const dim3 grid(unsigned((s.rows + chunk - 1) / chunk), unsigned(c.heads), 2);
    write_kernel<T, FMT><<<grid, W_CTA, 0, st>>>(static_cast<const T *>(k), ks, static_cast<const T *>(v), vs, c, s, chunk, packs_of_4<T>(k, ks, v, vs), flag);
}
template <typename T, int FMT>
void launch_read(const Cache &c, const Seqs &s, void *k, int64_t ks, void *v, int64_t vs, int32_t *flag, cudaStream_t st) {
    read_kernel<T, FMT><<<dim3(unsigned(s.rows), 2), W_CTA, 0, st>>>(c, s, static_cast<T *>(k), ks, static_cast<T *>(v), vs, packs_of_4<T>(k, ks, v, vs), flag);
}

}  // namespace
}  // namespace kv
}  // namespace dx

#define DX_KV_DISPATCH(CALL)                                                                         \
    switch (dtype * DX_CACHE_FORMAT_COUNT + cache->format) {                                         \
        case DX_F32 * DX_CACHE_FORMAT_COUNT + DX_CACHE_I8: CALL(float, DX_CACHE_I8); break;          \
        case DX_F32 * DX_CACHE_FORMAT_COUNT + DX_CACHE_E4M3: CALL(float, DX_CACHE_E4M3); break;      \
        case DX_F16 * DX_CACHE_FORMAT_COUNT + DX_CACHE_I8: CALL(f16, DX_CACHE_I8); break;            \
        case DX_F16 * DX_CACHE_FORMAT_COUNT + DX_CACHE_E4M3: CALL(f16, DX_CACHE_E4M3); break;        \
        case DX_BF16 * DX_CACHE_FORMAT_COUNT + DX_CACHE_I8: CALL(bf16, DX_CACHE_I8); break;          \
        default: CALL(bf16, DX_CACHE_E4M3); break;                                                   \
    }

extern "C" int dx_kvcache_write(int dtype, const void *k, int64_t k_stride, const void *v, int64_t v_stride, const dx_kvseqs *seqs,
                                const dx_kvcache *cache, int32_t *flag, void *stream) {
    using namespace dx;
    kv::Cache c;
    kv::Seqs s;
    if (int e = kv::check("kvcache_write", cache, seqs, &c, &s)) return e;
    if (int e = kv::check_rows("kvcache_write", dtype, s, c, k, k_stride, v, v_stride)) return e;
    if (s.rows == 0 || s.batch == 0) return DX_OK;
    cudaStream_t st = as_stream(stream);
#define DX_CALL(T, FMT) kv::launch_write<T, FMT>(k, k_stride, v, v_stride, c, s, flag, st)
    DX_KV_DISPATCH(DX_CALL)
#undef DX_CALL
    return check_launch("kvcache_write");
}

extern "C" int dx_kvcache_read(int dtype, const dx_kvseqs *seqs, const dx_kvcache *cache, void *k, int64_t k_stride, void *v, int64_t v_stride,
                               int32_t *flag, void *stream) {
    using namespace dx;
    kv::Cache c;
    kv::Seqs s;
    if (int e = kv::check("kvcache_read", cache, seqs, &c, &s)) return e;
    if (int e = kv::check_rows("kvcache_read", dtype, s, c, k, k_stride, v, v_stride)) return e;
    if (s.rows == 0 || s.batch == 0) return DX_OK;
    cudaStream_t st = as_stream(stream);
#define DX_CALL(T, FMT) kv::launch_read<T, FMT>(c, s, k, k_stride, v, v_stride, flag, st)
    DX_KV_DISPATCH(DX_CALL)
#undef DX_CALL
    return check_launch("kvcache_read");
}
