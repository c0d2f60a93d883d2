// What the kernels of dx_kvcache_attention share: the call's arguments, the parts of items that several blocks work on, and the
// kernel that joins them.
#pragma once
#include <atomic>

#include "kvcache.cuh"

namespace dx {
namespace kv {

struct Attn {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    int q_heads, group, window;
    float scale_log2;
    int q_vec, out_vec;  // 16-byte loads of q and stores of out are possible
    uint8_t *ws;
    int32_t *flag;
};

// What the joining kernel needs to know of the item that ends inside block i's first piece: `parts` blocks from i - 1 on hold
// parts of it (0: block i does not begin inside an item, or an earlier one joins it).
struct alignas(32) Join {
    int64_t row0;
    int first_row, rows, head, parts;
};

// Attention by tiles of 128 rows on the fifth-generation tensor cores (kvcache_tiles.cu), for head_dim up to 128.
size_t tiles_workspace(const Cache &c, const Seqs &s, int group);
int launch_tiles(int dtype, int format, const Attn &a, const Cache &c, const Seqs &s, cudaStream_t st);

// A kernel's shared memory above 48 KB has to be allowed once on each device.
template <typename F> int allow_shared(F *kernel, int bytes, std::atomic<uint64_t> *prepared) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (e == cudaSuccess && !(prepared->load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) prepared->fetch_or(bit, std::memory_order_relaxed);
    }
    return e == cudaSuccess ? DX_OK : fail(DX_E_CUDA, "kvcache_attention: %s", cudaGetErrorString(e));
}

#ifdef __CUDACC__
// A row's weights are 2^(x - m), x its scores in powers of two, m their running maximum, which may lag by LAG; their sum is one of 32-bit
// numbers.  What multiplies a value's code is the half of 2^(x - m) * s * 2^(7 - d), s the scale of the value's page and d the running maximum of
// x - m + log2(s), with the same lag: at most 2^15, and what is 2^-31 of the row's largest is still a half.  So a page that the row does not weigh
// takes no bits from the others, whatever its scale is.  Both are whole numbers (rounded up), and d is a small one where x is not: scores
// of any size are exact beside it.  Below D_LEAST no value is a normal number; a row begins there.
constexpr float LAG = 8.f, UP = 7.f, D_LEAST = -118.f, LOWEST = -3.402823466e38f;
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr int JOIN_CTA = 512;

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 2^x, off by 2^-22 of it; what is below 2^-126 becomes zero (without that, every call would be four instructions instead of one).
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The whole power of two that a scale is or lies below (for zero, one below all others).
__device__ __forceinline__ float scale_power(float s) {
    const uint32_t u = __float_as_uint(s) & 0x7FFFFFFFu;
    return __uint_as_float(0x4B000000u | (u + 0x7FFFFFu) >> 23) - (8388608.f + 127.f);  // the exponent without a conversion
}
// A row's running maxima.
struct Maxima {
    float m, d;
    __device__ __forceinline__ void clear() { m = LOWEST, d = D_LEAST; }
    // The row's largest score is `top`; top_v(m): its largest score less m with its scale's power.  How much the sum and the output so far are
    // in the new units.
    template <typename TopV> __device__ __forceinline__ void rise(float top, TopV top_v, float &of_sum, float &of_output) {
        const float to = top - m > LAG ? ceilf(top) : m;
        of_sum = to == m ? 1.f : exp2_approx(m - to);
        const float was = to == m ? d : d + (m - to);
        m = to;
        const float now = top_v(m);
        d = fmaxf(now > was + LAG ? ceilf(now) : was, D_LEAST);
        of_output = d == was ? 1.f : exp2_approx(was - d);
    }
};
__device__ __forceinline__ float or_zero(float m) { return m == NEG_INF ? 0.f : m; }
// What brings a row's output, in units of 2^(d - 7), over its sum to the result: output * first * second.  Two factors, as one could be out of
// float32's range where the result is not.
struct Out {
    float first, second;
};
__device__ __forceinline__ Out way_out(float d, float sum) {
    const float half = exp2_approx(0.5f * (d - UP));
    return {half, sum == 0.f ? 0.f : half / sum};
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Joins the parts of an item that several blocks worked on: each part's share of one from all parts' maxima and sums, then their outputs in the
// order of the keys.  A part is ROWS x DP floats of output, ROWS maxima and ROWS sums; block i's first piece leaves part 2i, one that begins
// with its item and does not end it part 2i + 1.  What it costs is waiting for memory, one load after the other, so there are two ways.
// Up to FEW parts: a warp takes a row (two where items have many) and has every load of it in flight at once, without waiting for a
// maximum.  (With the other way alone the join of 64 single tokens after 300 to 8192, 8 key heads of 128, took 13 us in place of 7, that
// of 2 x 4096 tokens, 32 heads, 30 in place of 14.)  More: sixteen warps take sixteen of the item's rows at a time, the warps of a row
// share its parts, and FLIGHT of a warp's parts are on their way at once.
__host__ __device__ constexpr int join_rows(int rows) { return rows > 128 ? 32 : 16; }  // of a block

template <typename T, int DP, int ROWS> __global__ void __launch_bounds__(JOIN_CTA, DP > 128 ? 1 : 2) join_kernel(Attn a, Cache c) {
    constexpr int V = DP / 32, VW = V < 4 ? V : 4, PART = ROWS * DP + 2 * ROWS, STEP = 16, FEW = 4;
    constexpr int FLIGHT = ROWS > 128 ? 2 : 8;
    __shared__ float sh[JOIN_CTA / 32][DP];
    griddep_wait_cta();
    const Join j = reinterpret_cast<const Join *>(a.ws)[blockIdx.x];
    const int first = blockIdx.y * join_rows(ROWS), last = min(j.rows, first + join_rows(ROWS));
    if (j.parts == 0 || first >= last) return;
    const float *parts = reinterpret_cast<const float *>(a.ws + gridDim.x * sizeof(Join));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto at = [&](int p) { return parts + (int64_t(blockIdx.x - 1 + p) * 2 + (p == 0 ? 1 : 0)) * PART; };
    auto out_row = [&](int row) {
        const int fr = j.first_row + row, i = fr / a.group;
        return static_cast<T *>(a.out) + (j.row0 + i) * a.out_stride + int64_t(j.head * a.group + fr - i * a.group) * c.dim;
    };
    if (j.parts <= FEW) {
        constexpr int EACH = join_rows(ROWS) / 16;
        Pack<float, VW> x[EACH][FEW][V / VW];
        float m[EACH][FEW], l[EACH][FEW];
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int row = first + k * 16 + warp;
#pragma unroll
            for (int p = 0; p < FEW; ++p) {
                m[k][p] = NEG_INF, l[k][p] = 0.f;
                if (row < last && p < j.parts) {
                    m[k][p] = at(p)[ROWS * DP + row];
                    l[k][p] = at(p)[ROWS * DP + ROWS + row];
#pragma unroll
                    for (int e = 0; e < V / VW; ++e) x[k][p][e] = reinterpret_cast<const Pack<float, VW> *>(at(p) + row * DP + lane * V)[e];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int row = first + k * 16 + warp;
            if (row >= last) continue;
            float top = m[k][0], sum = 0.f, acc[V] = {};
#pragma unroll
            for (int p = 1; p < FEW; ++p) top = fmaxf(top, m[k][p]);
            const float base = or_zero(top);
#pragma unroll
            for (int p = 0; p < FEW; ++p) sum += l[k][p] *= exp2_approx(m[k][p] - base);
            const float all = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int p = 0; p < FEW; ++p) {
                const float by = l[k][p] * all;  // shares of one: a sum that is divided afterwards could be out of range
                if (p < j.parts && by != 0.f)
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[e] += by * x[k][p][e / VW].v[e % VW];
            }
            T *out = out_row(row) + lane * V;
            if (lane * V >= c.dim) continue;  // dim is a multiple of 16, V a power of two up to 4: the lane's values are all of the row or none
            Pack<T, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) o.v[e] = from_compute<T>(acc[e]);
            if (reinterpret_cast<uintptr_t>(out) % sizeof(o) == 0) *reinterpret_cast<Pack<T, V> *>(out) = o;
            else
#pragma unroll
                for (int e = 0; e < V; ++e) out[e] = o.v[e];
        }
        return;
    }
#pragma unroll 1
    for (int row0 = first; row0 < last; row0 += STEP) {
        const int rows = min(last - row0, STEP);
        const int each = rows > 8 ? 1 : rows > 4 ? 2 : rows > 2 ? 4 : rows > 1 ? 8 : 16;  // warps of a row
        const int r = warp / each, row = row0 + r, sub = warp % each;
        float acc[V] = {};
        if (r < rows) {
            float top = NEG_INF, sum = 0.f;
            for (int p0 = lane; p0 < j.parts; p0 += 128) {
                float m[4], l[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = p0 + 32 * k < j.parts;
                    m[k] = in ? at(p0 + 32 * k)[ROWS * DP + row] : NEG_INF;
                    l[k] = in ? at(p0 + 32 * k)[ROWS * DP + ROWS + row] : 0.f;
                }
                const float to = fmaxf(top, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))), base = or_zero(to);
                sum *= exp2_approx(top - base);
                top = to;
#pragma unroll
                for (int k = 0; k < 4; ++k) sum += l[k] * exp2_approx(m[k] - base);
            }
            float most = top;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float base = or_zero(most);
            sum *= exp2_approx(top - base);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float all = sum == 0.f ? 0.f : 1.f / sum;
            for (int p0 = 0; p0 < j.parts; p0 += 32) {
                float w = 0.f;
                if (p0 + lane < j.parts) w = at(p0 + lane)[ROWS * DP + ROWS + row] * exp2_approx(at(p0 + lane)[ROWS * DP + row] - base) * all;
                const int n = min(32, j.parts - p0);
                for (int p1 = sub; p1 < n; p1 += FLIGHT * each) {
                    Pack<float, VW> x[FLIGHT][V / VW];
#pragma unroll
                    for (int k = 0; k < FLIGHT; ++k)
#pragma unroll
                        for (int e = 0; e < V / VW; ++e)
                            if (p1 + k * each < n) x[k][e] = reinterpret_cast<const Pack<float, VW> *>(at(p0 + p1 + k * each) + row * DP + lane * V)[e];
#pragma unroll
                    for (int k = 0; k < FLIGHT; ++k) {
                        const float by = __shfl_sync(0xffffffffu, w, min(p1 + k * each, 31));
                        if (p1 + k * each >= n || by == 0.f) continue;
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[e] += by * x[k][e / VW].v[e % VW];
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) sh[warp][lane * V + e] = acc[e];
        __syncthreads();
        if (r < rows && sub == 0) {
            T *out = out_row(row);
            for (int d = lane; d < c.dim; d += 32) {
                float v = 0.f;
                for (int w = 0; w < each; ++w) v += sh[warp + w][d];
                out[d] = from_compute<T>(v);
            }
        }
        __syncthreads();
    }
}
#endif

}  // namespace kv
}  // namespace dx
