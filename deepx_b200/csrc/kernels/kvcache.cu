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

constexpr int CTA = 256;
constexpr int MAX_CHUNK = 128;
constexpr int STARTS = 512;  // sequences whose starts a block copies into shared memory before it searches them

// Eight values of a row as they lie in memory.
template <typename T> struct Eight {
    static constexpr int N = 16 / sizeof(T), P = 8 / N;
    Pack<T, N> p[P];
    __device__ __forceinline__ void load(const T *x, bool vec) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (vec) p[i] = ld_cached<T, N>(x + i * N);
            else {
#pragma unroll
                for (int e = 0; e < N; ++e) p[i].v[e] = x[i * N + e];
            }
        }
    }
    __device__ __forceinline__ float get(int e) const { return to_compute(p[e / N].v[e % N]); }
};
// The larger of the sizes of eight values and `top`: not a number or infinite if one of them is.
template <typename T> __device__ __forceinline__ float size_of(const Eight<T> &x, float top) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int e = 0; e < 8; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x.get(e))));
        return top;
    } else {
        using T2 = typename std::conditional<std::is_same<T, f16>::value, __half2, __nv_bfloat162>::type;
        const T2 *v = reinterpret_cast<const T2 *>(x.p[0].v);
        const T2 m = __hmax2_nan(__hmax2_nan(__habs2(v[0]), __habs2(v[1])), __hmax2_nan(__habs2(v[2]), __habs2(v[3])));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(to_compute(m.x)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(to_compute(m.y)));
        return top;
    }
}
// The same of the finite ones among them.
template <typename T> __device__ __forceinline__ float finite_size_of(const Eight<T> &x, float top, bool &nan) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float f = fabsf(x.get(e));
        nan |= f != f;
        top = fmaxf(top, f < __int_as_float(0x7f800000) ? f : 0.f);
    }
    return top;
}
template <typename T, int FMT> __device__ __forceinline__ uint2 codes_of(const Eight<T> &x, float inv, bool finite) {
    if (finite) return make_uint2(encode4_finite<FMT>(x.get(0), x.get(1), x.get(2), x.get(3), inv), encode4_finite<FMT>(x.get(4), x.get(5), x.get(6), x.get(7), inv));
    return make_uint2(encode4<FMT>(x.get(0) * inv, x.get(1) * inv, x.get(2) * inv, x.get(3) * inv),
                      encode4<FMT>(x.get(4) * inv, x.get(5) * inv, x.get(6) * inv, x.get(7) * inv));
}
// The starts, copied into shared memory where they fit: a search is then one trip to memory instead of one for each halving.
__device__ __forceinline__ const int32_t *starts_near(const Seqs &s, int32_t *copy) {
    if (s.batch > STARTS) return s.starts;
    for (int i = threadIdx.x; i <= s.batch; i += CTA) copy[i] = s.starts[i];
    __syncthreads();
    return copy;
}

// A block takes the pages whose first new token is one of `chunk` packed rows, for one head: half of its threads the keys, half the
// values.  The page's values are loaded once: up to KEEP vectors of eight stay in a thread's registers between the search for
// their largest size and the rounding (a page of 64 tokens of 128 dimensions whole); the rest of larger pages is read again,
// out of the cache the first time has left it in.
template <typename T, int FMT, int KEEP>
__global__ void __launch_bounds__(CTA, 4) write_kernel(const T *k, int64_t k_stride, const T *v, int64_t v_stride, Cache c, Seqs s, int chunk,
                                                       FastDiv by_units, bool vec, int32_t *flag) {
    constexpr int SIDE = CTA / 2;
    struct Found {
        int64_t row;
        int b, pos, tokens;
    };
    __shared__ Found list[MAX_CHUNK];
    __shared__ int32_t copy[STARTS + 1];
    __shared__ int count;
    __shared__ float part[2][CTA / 32];
    griddep_wait_cta();
    const int side = threadIdx.x / SIDE, tid = threadIdx.x % SIDE, head = blockIdx.y;
    const T *x = side ? v : k;
    const int64_t stride = side ? v_stride : k_stride;
    uint8_t *codes = side ? c.v : c.k;
    float *scales = side ? c.v_scale : c.k_scale;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_seqs(s, c, flag);
    if (threadIdx.x == 0) count = 0;
    const int32_t *starts = starts_near(s, copy);
    __syncthreads();
    const int64_t row0 = int64_t(blockIdx.x) * chunk;
    if (int(threadIdx.x) < chunk && row0 + threadIdx.x < s.rows) {
        const int64_t row = row0 + threadIdx.x;
        const int b = seq_of_row(starts, s.batch, row);
        if (b >= 0) {
            const Seq q = seq_at(s, c, b);
            const int64_t i = row - q.row0;
            const int64_t pos = q.first + i;
            if (i >= 0 && i < q.n && pos >= 0 && pos < q.end && (i == 0 || pos == 0 || (pos & (c.page - 1)) == 0)) {
                const int room = min(c.page - int(pos & (c.page - 1)), q.end - int(pos));
                list[atomicAdd(&count, 1)] = Found{row, b, int(pos), int(min(int64_t(room), q.n - i))};
            }
        }
    }
    __syncthreads();
    const int units = c.dim / 8, found = count;
    for (int n = 0; n < found; ++n) {
        const Found f = list[n];
        const int slot = f.pos & (c.page - 1), total = f.tokens * units;
        const int64_t page = page_at(s, c, f.b, f.pos, threadIdx.x == 0 ? flag : nullptr);
        if (page < 0) continue;  // the same answer in every thread
        const T *src = x + f.row * stride + int64_t(head) * c.dim;
        uint8_t *dst = codes + ((page * c.heads + head) * c.page) * int64_t(c.dim);
        float *scale_at = scales + page * c.heads + head;
        const float had = slot ? *scale_at : 0.f;
        auto at = [&](int u) {
            const int t = int(fd_div(uint32_t(u), by_units));
            return src + t * stride + (u - t * units) * 8;
        };
        Eight<T> kept[KEEP];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (tid + i * SIDE < total) kept[i].load(at(tid + i * SIDE), vec);
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (tid + i * SIDE < total) amax = size_of(kept[i], amax);
        for (int u = tid + KEEP * SIDE; u < total; u += SIDE) {
            Eight<T> more;
            more.load(at(u), vec);
            amax = size_of(more, amax);
        }
        const bool finite = amax < __int_as_float(0x7f800000);  // of this thread's values
        bool nan = false;
        if (!finite) {
            amax = 0.f;
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
                if (tid + i * SIDE < total) amax = finite_size_of(kept[i], amax, nan);
            for (int u = tid + KEEP * SIDE; u < total; u += SIDE) {
                Eight<T> more;
                more.load(at(u), vec);
                amax = finite_size_of(more, amax, nan);
            }
        }
        if (nan) raise(flag, FLAG_NAN);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((threadIdx.x & 31) == 0) part[n & 1][threadIdx.x >> 5] = amax;
        __syncthreads();  // and every thread has read the old scale
#pragma unroll
        for (int w = 0; w < SIDE / 32; ++w) amax = fmaxf(amax, part[n & 1][side * (SIDE / 32) + w]);
        float scale = scale_for<FMT>(amax);
        if (slot) scale = fmaxf(scale, scale_kept(had));
        const float inv = inverse_of(scale);
        if (slot && scale != had) {  // the earlier tokens' codes in units of the grown scale
            const float by = had * inv;
            for (int u = tid; u < slot * units; u += SIDE) {
                uint2 w = *reinterpret_cast<const uint2 *>(dst + int64_t(u) * 8);
                for (uint32_t *e : {&w.x, &w.y}) {
                    const float2 lo = __half22float2(decode2<FMT>(*e & 0xFFFFu)), hi = __half22float2(decode2<FMT>(*e >> 16));
                    *e = encode4<FMT>(lo.x * by, lo.y * by, hi.x * by, hi.y * by);
                }
                *reinterpret_cast<uint2 *>(dst + int64_t(u) * 8) = w;
            }
        }
        uint2 *out = reinterpret_cast<uint2 *>(dst) + int64_t(slot) * units;
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (tid + i * SIDE < total) out[tid + i * SIDE] = codes_of<T, FMT>(kept[i], inv, finite);
        for (int u = tid + KEEP * SIDE; u < total; u += SIDE) {
            Eight<T> more;
            more.load(at(u), vec);
            out[u] = codes_of<T, FMT>(more, inv, finite);
        }
        if (tid == 0) *scale_at = scale;
    }
}

// A block takes `chunk` packed rows: where each one's codes are is worked out once, then sixteen codes (one 16-byte load) a thread and
// turn, keys and values in one go.
template <typename T, int FMT>
__global__ void __launch_bounds__(CTA) read_kernel(Cache c, Seqs s, T *k, int64_t k_stride, T *v, int64_t v_stride, int chunk, FastDiv by_row,
                                                   FastDiv by_units, bool vec, int32_t *flag) {
    constexpr int N = 16 / sizeof(T);
    constexpr int64_t NONE = -1, ZERO = -2;
    __shared__ int64_t page_of[MAX_CHUNK];  // page number, or NONE: no sequence's row, ZERO: no token's
    __shared__ int slot_of[MAX_CHUNK];
    __shared__ int32_t copy[STARTS + 1];
    griddep_wait_cta();
    if (blockIdx.x == 0) check_seqs(s, c, flag);
    const int32_t *starts = starts_near(s, copy);
    const int64_t row0 = int64_t(blockIdx.x) * chunk;
    const int rows = int(min(int64_t(chunk), s.rows - row0));
    if (int(threadIdx.x) < rows) {
        const int64_t row = row0 + threadIdx.x;
        const int b = seq_of_row(starts, s.batch, row);
        int64_t page = NONE;
        if (b >= 0) {
            const Seq q = seq_at(s, c, b);
            const int64_t i = row - q.row0, pos = q.first + i;
            if (i >= 0 && i < q.n) {
                page = ZERO;
                if (pos >= 0 && pos < q.end) {
                    page = page_at(s, c, b, int(pos), flag);
                    if (page < 0) page = ZERO;
                    slot_of[threadIdx.x] = int(pos & (c.page - 1));
                }
            }
        }
        page_of[threadIdx.x] = page;
    }
    __syncthreads();
    const int units = c.dim / 16, per_row = c.heads * units;
    for (int i = threadIdx.x; i < 2 * rows * per_row; i += CTA) {
        const int line = int(fd_div(uint32_t(i), by_row)), u = i - line * per_row, r = line >> 1;  // a row's keys, then its values
        const bool is_v = line & 1;
        const int64_t page = page_of[r];
        if (page == NONE) continue;
        T *out = (is_v ? v + (row0 + r) * v_stride : k + (row0 + r) * k_stride) + int64_t(u) * 16;
        uint4 w = make_uint4(0, 0, 0, 0);
        float f = 0.f;
        if (page >= 0) {
            const int h = int(fd_div(uint32_t(u), by_units));
            const int64_t ph = page * c.heads + h;
            w = __ldcs(reinterpret_cast<const uint4 *>((is_v ? c.v : c.k) + (ph * c.page + slot_of[r]) * c.dim + (u - h * units) * 16));
            f = (is_v ? c.v_scale : c.k_scale)[ph];
        }
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        Pack<T, N> o[16 / N];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 lo = __half22float2(decode2<FMT>(words[e] & 0xFFFFu)), hi = __half22float2(decode2<FMT>(words[e] >> 16));
            const float x[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
            for (int d = 0; d < 4; ++d) o[(4 * e + d) / N].v[(4 * e + d) % N] = from_compute<T>(x[d] * f);
        }
#pragma unroll
        for (int p = 0; p < 16 / N; ++p) {
            if (vec) st_stream<T, N>(out + p * N, o[p]);
            else {
#pragma unroll
                for (int e = 0; e < N; ++e) out[p * N + e] = o[p].v[e];
            }
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

template <typename T> bool vectors(const void *k, int64_t k_stride, const void *v, int64_t v_stride) {
    constexpr int N = 16 / sizeof(T);
    return k_stride % N == 0 && v_stride % N == 0 && aligned_to(k, 16) && aligned_to(v, 16);
}

template <typename T, int FMT>
void launch_write(const void *k, int64_t ks, const void *v, int64_t vs, const Cache &c, const Seqs &s, int32_t *flag, cudaStream_t st) {
    // rows a block searches for first tokens of pages: one for single tokens, a page's worth for prompts
    int chunk = 1;
    while (chunk < MAX_CHUNK && chunk < c.page && int64_t(chunk) * s.batch < s.rows) chunk *= 2;
    const dim3 grid(unsigned((s.rows + chunk - 1) / chunk), unsigned(c.heads));
    const bool vec = vectors<T>(k, ks, v, vs);
    if (chunk == 1) launch_pdl(write_kernel<T, FMT, 1>, grid, dim3(CTA), 0, st, static_cast<const T *>(k), ks, static_cast<const T *>(v), vs, c, s, chunk, make_fastdiv(c.dim / 8), vec, flag);
    else launch_pdl(write_kernel<T, FMT, 8>, grid, dim3(CTA), 0, st, static_cast<const T *>(k), ks, static_cast<const T *>(v), vs, c, s, chunk, make_fastdiv(c.dim / 8), vec, flag);
}
template <typename T, int FMT>
void launch_read(const Cache &c, const Seqs &s, void *k, int64_t ks, void *v, int64_t vs, int32_t *flag, cudaStream_t st) {
    int chunk = 1;
    while (chunk < 16 && s.rows > int64_t(sm_count()) * 8 * chunk) chunk *= 2;
    launch_pdl(read_kernel<T, FMT>, dim3(unsigned((s.rows + chunk - 1) / chunk)), dim3(CTA), 0, st, c, s, static_cast<T *>(k), ks, static_cast<T *>(v), vs, chunk,
               make_fastdiv(unsigned(c.heads * (c.dim / 16))), make_fastdiv(c.dim / 16), vectors<T>(k, ks, v, vs), flag);
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
