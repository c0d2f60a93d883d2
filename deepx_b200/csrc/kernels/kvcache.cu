// dx_kvcache_write and dx_kvcache_read: values into the pages of an 8-bit key/value cache, and back.
//
// Both are bound by memory: a value is read (written) once at its type's size, its code written (read) once.  Measured (B200): writing four
// prompts of 5000 to 8192 tokens, 8 heads of 128, bf16 to e4m3: 37.3 us, 4.6 TB/s of the copy's 6.5; reading eight histories of 3000 to
// 9000 tokens, 8 heads of 64, e4m3 to f16: 32.2 us, 4.7 TB/s.  Sixteen values a thread, moved 32 bytes at a time where the rows allow it
// (eight at 16 bytes: 41 and 35 us); 64 single tokens: 3.6 us on the device, a launch's latency.
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

constexpr int CTA = 256;   // of the kernel that reads
constexpr int SIDE = 128;  // of the kernel that writes, and how many of its blocks an SM holds
constexpr int BLKS = 7;
constexpr int MAX_CHUNK = 128;
constexpr int STARTS = 512;  // sequences whose starts a block copies into shared memory before it searches them

// How a row's values can be moved: 32 bytes at a time, 16, or one value at a time.
enum Width : int { ONE = 0, W16 = 1, W32 = 2 };

// Sixteen values of a row as they lie in memory.
template <typename T> struct Sixteen {
    static constexpr int WORDS = 16 * sizeof(T) / 4;
    union {
        uint32_t w[WORDS];
        T v[16];
    };
    __device__ __forceinline__ Sixteen() {}
    __device__ __forceinline__ void load(const T *x, int width) {
        if (width == W32) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 8)
                asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                             : "l"(reinterpret_cast<const uint32_t *>(x) + i));
        } else if (width == W16) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 q = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(x) + i);
                w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = x[e];
        }
    }
    __device__ __forceinline__ void store(T *x, int width) const {
        if (width == W32) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 8)
                asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]),
                             "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7]), "l"(reinterpret_cast<uint32_t *>(x) + i)
                             : "memory");
        } else if (width == W16) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) __stcs(reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(x) + i), make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]));
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = v[e];
        }
    }
    __device__ __forceinline__ void set4(int i, float a, float b, float c, float d) {  // values 4i.., two at a time: one conversion
        if constexpr (std::is_same<T, bf16>::value) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
            w[2 * i] = *reinterpret_cast<const uint32_t *>(&x), w[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&y);
        } else if constexpr (std::is_same<T, f16>::value) {
            const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
            w[2 * i] = *reinterpret_cast<const uint32_t *>(&x), w[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&y);
        } else {
            w[4 * i] = __float_as_uint(a), w[4 * i + 1] = __float_as_uint(b), w[4 * i + 2] = __float_as_uint(c), w[4 * i + 3] = __float_as_uint(d);
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else if constexpr (std::is_same<T, bf16>::value) return __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
        else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e >> 1]));
            return e & 1 ? f.y : f.x;
        }
    }
};
// The larger of the sizes of sixteen values and `top`: not a number or infinite if one of them is.
template <typename T> __device__ __forceinline__ float size_of(const Sixteen<T> &x, float top) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int e = 0; e < 16; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x.get(e))));
    } else {
        using T2 = typename std::conditional<std::is_same<T, f16>::value, __half2, __nv_bfloat162>::type;
        T2 m = __habs2(*reinterpret_cast<const T2 *>(&x.w[0]));
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const T2 *>(&x.w[i])));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(to_compute(m.x)));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(to_compute(m.y)));
    }
    return top;
}
// The same of the finite ones among them.
template <typename T> __device__ __forceinline__ float finite_size_of(const Sixteen<T> &x, float top, bool &nan) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float f = fabsf(x.get(e));
        nan |= f != f;
        top = fmaxf(top, f < __int_as_float(0x7f800000) ? f : 0.f);
    }
    return top;
}
template <typename T, int FMT> __device__ __forceinline__ uint4 codes_of(const Sixteen<T> &x, float inv, bool finite) {
    uint32_t c[4];
    if (finite) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = encode4_finite<FMT>(x.get(4 * i), x.get(4 * i + 1), x.get(4 * i + 2), x.get(4 * i + 3), inv);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = encode4<FMT>(x.get(4 * i) * inv, x.get(4 * i + 1) * inv, x.get(4 * i + 2) * inv, x.get(4 * i + 3) * inv);
    }
    return make_uint4(c[0], c[1], c[2], c[3]);
}
// The starts, copied into shared memory where they fit: a search is then one trip to memory instead of one for each halving.
__device__ __forceinline__ const int32_t *starts_near(const Seqs &s, int32_t *copy) {
    if (s.batch > STARTS) return s.starts;
    for (int i = threadIdx.x; i <= s.batch; i += blockDim.x) copy[i] = s.starts[i];
    __syncthreads();
    return copy;
}

// A block takes the pages whose first new token is one of `chunk` packed rows, for `head_count` heads one after the other, and of them the
// keys or the values.  A page's values are loaded once: up to KEEP pieces of sixteen stay in a thread's registers between the search for
// their largest size and the rounding (a page of 64 tokens of 128 dimensions whole, in 16 bits); the rest of larger pages is read again, out
// of the cache the first time has left it in.  Every unit of a page and a head waits for memory, then for its block's largest value, then
// rounds: what hides that is other blocks, so blocks are small (seven of 128 threads an SM; three of 256 with keys and values in one
// measured 38.5 us in place of 37.3 for four prompts of 5000 to 8192 tokens, 8 heads of 128, bf16).
template <typename T, int FMT, int KEEP>
__global__ void __launch_bounds__(SIDE, BLKS) write_kernel(const T *k, int64_t k_stride, const T *v, int64_t v_stride, Cache c, Seqs s, int chunk,
                                                       int head_count, int width, int32_t *flag) {
    struct Found {
        int64_t row;
        int b, pos, tokens;
    };
    __shared__ Found list[MAX_CHUNK];
    __shared__ int32_t copy[STARTS + 1];
    __shared__ int count;
    __shared__ float part[2][SIDE / 32];
    griddep_wait_cta();
    const int side = blockIdx.z, tid = threadIdx.x;
    const T *x = side ? v : k;
    const int64_t stride = side ? v_stride : k_stride;
    uint8_t *codes = side ? c.v : c.k;
    float *scales = side ? c.v_scale : c.k_scale;
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) check_seqs(s, c, flag);
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
    // a thread takes sixteen columns of every pass_rows-th token (the threads behind the last whole row of a pass have none)
    const int units = c.dim / 16, found = count, pass_rows = SIDE / units, row_in = tid / units, col = (tid - row_in * units) * 16;
    const int64_t pass = pass_rows * stride;
    const int pass_codes = pass_rows * c.dim, head0 = blockIdx.y * head_count, head1 = min(head0 + head_count, c.heads);
    int turn = 0;
    for (int n = 0; n < found; ++n) {
        const Found f = list[n];
        const int slot = f.pos & (c.page - 1), rows = row_in < pass_rows ? f.tokens : 0;  // of this thread's columns
        const int64_t page = page_at(s, c, f.b, f.pos, threadIdx.x == 0 ? flag : nullptr);
        if (page < 0) continue;  // the same answer in every thread
        const T *mine = x + (f.row + row_in) * stride + int64_t(head0) * c.dim + col;
        uint8_t *page_at0 = codes + ((page * c.heads + head0) * c.page) * int64_t(c.dim);
        float *scale_at = scales + page * c.heads + head0;
        for (int head = head0; head < head1; ++head, mine += c.dim, page_at0 += c.page * c.dim, ++scale_at, turn ^= 1) {
            const float had = slot ? *scale_at : 0.f;
            Sixteen<T> kept[KEEP];
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
                if (row_in + i * pass_rows < rows) kept[i].load(mine + i * pass, width);
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
                if (row_in + i * pass_rows < rows) amax = size_of(kept[i], amax);
#pragma unroll 1
            for (int i = KEEP; row_in + i * pass_rows < rows; ++i) {
                Sixteen<T> more;
                more.load(mine + i * pass, width);
                amax = size_of(more, amax);
            }
            const bool finite = amax < __int_as_float(0x7f800000);  // of this thread's values
            bool nan = false;
            if (!finite) {
                amax = 0.f;
#pragma unroll 1
                for (int i = 0; row_in + i * pass_rows < rows; ++i) {
                    Sixteen<T> more;
                    more.load(mine + i * pass, width);
                    amax = finite_size_of(more, amax, nan);
                }
            }
            if (nan) raise(flag, FLAG_NAN);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = amax;
            __syncthreads();  // and every thread has read the old scale
#pragma unroll
            for (int w = 0; w < SIDE / 32; ++w) amax = fmaxf(amax, part[turn][w]);
            float scale = scale_for<FMT>(amax);
            if (slot) scale = fmaxf(scale, scale_kept(had));
            const float inv = inverse_of(scale);
            if (slot && scale != had) {  // the earlier tokens' codes in units of the grown scale
                const float by = had * inv;
#pragma unroll 1
                for (int u = tid; u < slot * (c.dim / 8); u += SIDE) {
                    uint2 w = *reinterpret_cast<const uint2 *>(page_at0 + int64_t(u) * 8);
                    for (uint32_t *e : {&w.x, &w.y}) {
                        const float2 lo = __half22float2(decode2<FMT>(*e & 0xFFFFu)), hi = __half22float2(decode2<FMT>(*e >> 16));
                        *e = encode4<FMT>(lo.x * by, lo.y * by, hi.x * by, hi.y * by);
                    }
                    *reinterpret_cast<uint2 *>(page_at0 + int64_t(u) * 8) = w;
                }
            }
            uint8_t *out = page_at0 + (slot + row_in) * c.dim + col;
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
                if (row_in + i * pass_rows < rows) *reinterpret_cast<uint4 *>(out + i * pass_codes) = codes_of<T, FMT>(kept[i], inv, finite);
#pragma unroll 1
            for (int i = KEEP; row_in + i * pass_rows < rows; ++i) {
                Sixteen<T> more;
                more.load(mine + i * pass, width);
                *reinterpret_cast<uint4 *>(out + i * pass_codes) = codes_of<T, FMT>(more, inv, finite);
            }
            if (tid == 0) *scale_at = scale;
        }
    }
}

// A block takes `chunk` packed rows: where each one's codes are is worked out once, then sixteen codes (one 16-byte load) a thread and
// turn, keys and values in one go, stored 32 bytes at a time.
template <typename T, int FMT>
__global__ void __launch_bounds__(CTA) read_kernel(Cache c, Seqs s, T *k, int64_t k_stride, T *v, int64_t v_stride, int chunk, FastDiv by_row,
                                                   FastDiv by_units, int width, int32_t *flag) {
    constexpr int64_t NONE = -1, ZERO = -2;
    __shared__ int64_t code_of[MAX_CHUNK], scale_of[MAX_CHUNK];  // where a row's codes and scales begin, or NONE: no sequence's row, ZERO: no token's
    __shared__ int32_t copy[STARTS + 1];
    griddep_wait_cta();
    if (blockIdx.x == 0) check_seqs(s, c, flag);
    const int32_t *starts = starts_near(s, copy);
    const int64_t row0 = int64_t(blockIdx.x) * chunk;
    const int rows = int(min(int64_t(chunk), s.rows - row0));
    if (int(threadIdx.x) < rows) {
        const int64_t row = row0 + threadIdx.x;
        const int b = seq_of_row(starts, s.batch, row);
        int64_t at = NONE;
        if (b >= 0) {
            const Seq q = seq_at(s, c, b);
            const int64_t i = row - q.row0, pos = q.first + i;
            if (i >= 0 && i < q.n) {
                at = ZERO;
                const int64_t page = pos >= 0 && pos < q.end ? page_at(s, c, b, int(pos), flag) : -1;
                if (page >= 0) {
                    at = (page * c.heads * c.page + (pos & (c.page - 1))) * c.dim;
                    scale_of[threadIdx.x] = page * c.heads;
                }
            }
        }
        code_of[threadIdx.x] = at;
    }
    __syncthreads();
    const int units = c.dim / 16, per_row = c.heads * units;
    const int64_t next_head = int64_t(c.page - 1) * c.dim;  // a head's codes of a slot lie a page further than the head's before
#pragma unroll 2
    for (int i = threadIdx.x; i < 2 * rows * per_row; i += CTA) {
        const int line = int(fd_div(uint32_t(i), by_row)), u = i - line * per_row, r = line >> 1;  // a row's keys, then its values
        const bool is_v = line & 1;
        const int64_t at = code_of[r];
        if (at == NONE) continue;
        uint4 w = make_uint4(0, 0, 0, 0);
        float f = 0.f;
        if (at >= 0) {
            const int h = int(fd_div(uint32_t(u), by_units));
            w = __ldcs(reinterpret_cast<const uint4 *>((is_v ? c.v : c.k) + (at + u * 16 + h * next_head)));
            f = (is_v ? c.v_scale : c.k_scale)[scale_of[r] + h];
        }
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        Sixteen<T> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 lo = __half22float2(decode2<FMT>(words[e] & 0xFFFFu)), hi = __half22float2(decode2<FMT>(words[e] >> 16));
            o.set4(e, lo.x * f, lo.y * f, hi.x * f, hi.y * f);
        }
        o.store((is_v ? v + (row0 + r) * v_stride : k + (row0 + r) * k_stride) + int64_t(u) * 16, width);
    }
}

// What both entries check of their rows and of what their memory shares; `write`: the rows are read and the cache written, else the other way round.
int check_rows(const char *what, bool write, int dtype, const Seqs &s, const Cache &c, const void *k, int64_t k_stride, const void *v, int64_t v_stride, const int32_t *flag) {
    if (dtype != DX_F32 && dtype != DX_F16 && dtype != DX_BF16) return fail(DX_E_DTYPE, "%s: unsupported dtype code %d (float32, float16, bfloat16)", what, dtype);
    const int64_t width = int64_t(c.heads) * c.dim;
    if (k_stride < width || v_stride < width) return fail(DX_E_SHAPE, "%s: rows of %lld elements overlap at strides %lld and %lld", what, (long long)width, (long long)k_stride, (long long)v_stride);
    if (s.rows == 0 || s.batch == 0) return DX_OK;
    if (!k || !v) return fail(DX_E_ARG, "%s: null tensor pointer", what);
    const int64_t es = dx_dtype_size(dtype);
    const Span rows[2] = {span(k, s.rows, k_stride * es, width * es), span(v, s.rows, v_stride * es, width * es)}, raised = span(flag, 4);
    const CacheSpans cache(c, s);
    for (const Span &x : rows)
        if (meet(x, cache.codes[0]) || meet(x, cache.codes[1]) || meet(x, cache.scales[0]) || meet(x, cache.scales[1])) return fail(DX_E_ALIAS, "%s: a tensor overlaps the cache", what);
    if (!write && (meet(rows[0], rows[1]) || cache.lists_met_by(rows[0]) || cache.lists_met_by(rows[1])))
        return fail(DX_E_ALIAS, "%s: an output overlaps the other one or starts, lens or table", what);
    if (write) {
        const Span *out[4] = {&cache.codes[0], &cache.codes[1], &cache.scales[0], &cache.scales[1]};
        for (int i = 0; i < 4; ++i) {
            if (cache.lists_met_by(*out[i])) return fail(DX_E_ALIAS, "%s: the cache overlaps starts, lens or table", what);
            for (int n = 0; n < i; ++n)
                if (meet(*out[i], *out[n])) return fail(DX_E_ALIAS, "%s: the cache's tensors overlap", what);
        }
    }
    if (cache.met_by(raised) || meet(rows[0], raised) || meet(rows[1], raised)) return fail(DX_E_ALIAS, "%s: the flag lies in a tensor", what);
    return DX_OK;
}

template <typename T> int width_of(const void *k, int64_t k_stride, const void *v, int64_t v_stride) {
    for (int bytes : {32, 16}) {
        const int n = bytes / int(sizeof(T));
        if (k_stride % n == 0 && v_stride % n == 0 && aligned_to(k, bytes) && aligned_to(v, bytes)) return bytes == 32 ? W32 : W16;
    }
    return ONE;
}

template <typename T, int FMT>
void launch_write(const void *k, int64_t ks, const void *v, int64_t vs, const Cache &c, const Seqs &s, int32_t *flag, cudaStream_t st) {
    // rows a block searches for first tokens of pages: one for single tokens, a page's worth for prompts
    int chunk = 1;
    while (chunk < MAX_CHUNK && chunk < c.page && int64_t(chunk) * s.batch < s.rows) chunk *= 2;
    const int64_t blocks = (s.rows + chunk - 1) / chunk;
    // heads a block takes one after the other, so that the search is worth it: as many as leave every SM eight blocks
    int head_count = 1;
    while (head_count < 4 && blocks * ((c.heads + 2 * head_count - 1) / (2 * head_count)) >= int64_t(sm_count()) * 8) head_count *= 2;
    const dim3 grid(unsigned(blocks), unsigned((c.heads + head_count - 1) / head_count), 2);
    constexpr int KEEP = sizeof(T) == 4 ? 2 : 4;
    const int width = width_of<T>(k, ks, v, vs);
    if (chunk == 1) launch_pdl(write_kernel<T, FMT, 1>, grid, dim3(SIDE), 0, st, static_cast<const T *>(k), ks, static_cast<const T *>(v), vs, c, s, chunk, head_count, width, flag);
    else launch_pdl(write_kernel<T, FMT, KEEP>, grid, dim3(SIDE), 0, st, static_cast<const T *>(k), ks, static_cast<const T *>(v), vs, c, s, chunk, head_count, width, flag);
}
template <typename T, int FMT>
void launch_read(const Cache &c, const Seqs &s, void *k, int64_t ks, void *v, int64_t vs, int32_t *flag, cudaStream_t st) {
    int chunk = 1;  // rows of a block: up to 16 (with 32 or 64 the case above takes 34 and 35 us)
    while (chunk < 16 && s.rows > int64_t(sm_count()) * 8 * chunk) chunk *= 2;
    launch_pdl(read_kernel<T, FMT>, dim3(unsigned((s.rows + chunk - 1) / chunk)), dim3(CTA), 0, st, c, s, static_cast<T *>(k), ks, static_cast<T *>(v), vs, chunk,
               make_fastdiv(unsigned(c.heads * (c.dim / 16))), make_fastdiv(c.dim / 16), width_of<T>(k, ks, v, vs), flag);
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
    if (int e = kv::check_rows("kvcache_write", true, dtype, s, c, k, k_stride, v, v_stride, flag)) return e;
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
    if (int e = kv::check_rows("kvcache_read", false, dtype, s, c, k, k_stride, v, v_stride, flag)) return e;
    if (s.rows == 0 || s.batch == 0) return DX_OK;
    cudaStream_t st = as_stream(stream);
#define DX_CALL(T, FMT) kv::launch_read<T, FMT>(c, s, k, k_stride, v, v_stride, flag, st)
    DX_KV_DISPATCH(DX_CALL)
#undef DX_CALL
    return check_launch("kvcache_read");
}
