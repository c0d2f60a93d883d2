// What the kernels around the 8-bit key/value cache share: how a call's sequences and pages are found on the device, and
// how values become codes and codes values.
//
// Pages hold `page` tokens of `heads` key heads: [pages][heads][page][dim] codes of 8 bits, and one scale for each page and
// head.  A value stands for code * scale.  Scales are powers of two: dividing by one is exact, so a code depends on the
// value and the exponent alone, codes that are rounded again after a scale has grown lose at most another half step (e4m3
// codes nothing, down to the format's smallest), and code * scale is exact in every float type.  An arbitrary scale would
// use up to one bit more of an int8 code, and lose it again when pages are filled token by token.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace dx {
namespace kv {

constexpr int MAX_DIM = 256;
enum Flag : int { FLAG_PAGE = 1, FLAG_SEQS = 2, FLAG_NAN = 4 };

struct Cache {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    int64_t pages;
    int heads, page, page_shift, dim;
};
struct Seqs {
    const int32_t *starts, *lens, *table;
    int batch, cols;
    int64_t rows;
};

// Checks of the two descriptors that every entry point makes; DX_OK, or the code `fail` returned.
int check(const char *what, const dx_kvcache *c, const dx_kvseqs *s, Cache *cache, Seqs *seqs);
// The memory that the descriptors name.
struct CacheSpans {
    Span codes[2], scales[2], lists[3];
    CacheSpans(const Cache &c, const Seqs &s) {
        const int64_t n = c.pages * c.heads, bytes = n * c.page * c.dim;
        codes[0] = span(c.k, bytes), codes[1] = span(c.v, bytes), scales[0] = span(c.k_scale, n * 4), scales[1] = span(c.v_scale, n * 4);
        lists[0] = span(s.starts, (int64_t(s.batch) + 1) * 4), lists[1] = span(s.lens, int64_t(s.batch) * 4);
        lists[2] = span(s.table, int64_t(s.batch) * s.cols * 4);
    }
    bool met_by(const Span &x) const {
        for (int i = 0; i < 2; ++i)
            if (meet(x, codes[i]) || meet(x, scales[i])) return true;
        return lists_met_by(x);
    }
    bool lists_met_by(const Span &x) const { return meet(x, lists[0]) || meet(x, lists[1]) || meet(x, lists[2]); }
};

#ifdef __CUDACC__
__device__ __forceinline__ void raise(int32_t *flag, int bit) {
    if (flag) atomicOr(flag, bit);
}

// One sequence of the call.  `first` is the position of its first new token (negative when more new tokens are named than
// the sequence holds: those in front of position 0 do not exist), `end` how many tokens its pages can be read for.
struct Seq {
    int64_t row0;
    int n, first, end;
};
__device__ __forceinline__ Seq seq_at(const Seqs &s, const Cache &c, int b) {
    const int64_t s0 = s.starts[b], s1 = s.starts[b + 1], len = max(s.lens[b], 0);
    Seq r;
    r.row0 = max(s0, int64_t(0));
    const int64_t last = min(s1, s.rows);
    r.n = last > r.row0 ? int(last - r.row0) : 0;
    r.first = int(max(len - max(s1 - s0, int64_t(0)) + (r.row0 - s0), -(int64_t(1) << 31)));
    r.end = int(min(len, int64_t(s.cols) << c.page_shift));
    return r;
}
// Starts that do not ascend inside the packed rows, and lengths that the table cannot hold, raise a flag: what there is of
// them is worked on, nothing out of range is touched.  Called by one block of a launch, by all its threads.
__device__ __forceinline__ void check_seqs(const Seqs &s, const Cache &c, int32_t *flag) {
    if (!flag) return;
    bool bad = false;
    for (int b = threadIdx.x; b < s.batch; b += blockDim.x)
        bad |= s.starts[b] < 0 || s.starts[b + 1] < s.starts[b] || s.starts[b + 1] > s.rows || s.lens[b] < 0 ||
               s.lens[b] > (int64_t(s.cols) << c.page_shift);
    if (bad) raise(flag, FLAG_SEQS);
}
// The sequence that packed row `row` is a new token of, or -1.  `starts` may be a copy in shared memory.
__device__ __forceinline__ int seq_of_row(const int32_t *starts, int batch, int64_t row) {
    int lo = 0, hi = batch + 1;  // the last b with starts[b] <= row: of several sequences that start there the one that is not empty
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= row) lo = mid + 1;
        else hi = mid;
    }
    return lo - 1 < batch ? lo - 1 : -1;
}
// The page that holds position `pos` of sequence b (pos < end), or -1 and a flag when its number is none of the cache's.
__device__ __forceinline__ int64_t page_at(const Seqs &s, const Cache &c, int b, int pos, int32_t *flag) {
    const int64_t p = s.table[int64_t(b) * s.cols + (pos >> c.page_shift)];
    if (p >= 0 && p < c.pages) return p;
    raise(flag, FLAG_PAGE);
    return -1;
}

template <int FMT> struct Code;
// The least power of two, 2^-126 at least, in whose units `amax` is within the codes' range.  QMAX = TOP * 2^EXP in binary.
template <int FMT> __device__ __forceinline__ float scale_for(float amax) {
    constexpr uint32_t top = FMT == DX_CACHE_I8 ? 0x7E0000u : 0x600000u;  // 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
    constexpr int exp = FMT == DX_CACHE_I8 ? 6 : 8;
    const uint32_t u = __float_as_uint(amax);
    const int e = int(u >> 23) - 127 - exp + ((u & 0x7FFFFFu) > top ? 1 : 0);
    return __uint_as_float(uint32_t(max(e, -126) + 127) << 23);
}
// A scale that a page has already, as a power of two (what is no positive number counts as none).
__device__ __forceinline__ float scale_kept(float s) {
    if (!(s > 0.f && s < __int_as_float(0x7f800000))) return __uint_as_float(1u << 23);
    const uint32_t u = __float_as_uint(s);
    const uint32_t e = (u >> 23) + ((u & 0x7FFFFFu) ? 1 : 0);
    return __uint_as_float(min(max(e, 1u), 254u) << 23);
}
// 1/s of a power of two s in [2^-126, 2^127]; 2^-127 is no normal number, the only one that is rounded (to 2^-126: codes of
// values near the end of float32's range).
__device__ __forceinline__ float inverse_of(float s) {
    return __uint_as_float(max(254u - (__float_as_uint(s) >> 23), 1u) << 23);
}

// Four values in units of their scale → four codes, the first in the lowest byte.  Not a number becomes 0.
template <int FMT> __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (FMT == DX_CACHE_I8) {
        auto one = [](float x) {
            x = x == x ? fminf(fmaxf(x, -127.f), 127.f) : 0.f;
            return uint32_t(__float2int_rn(x)) & 0xFFu;
        };
        return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
    } else {
        auto fix = [](float x) { return x == x ? x : 0.f; };
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(fix(a), fix(b)), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(fix(c), fix(d)), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}
// The same of finite values within the codes' range, times `inv`, a power of two: for int8 one fused multiply-add rounds a value to a
// whole number in the low bits of a float (ties to even, as the unit of 1.5 * 2^23 is 1).
template <int FMT> __device__ __forceinline__ uint32_t encode4_finite(float a, float b, float c, float d, float inv) {
    if constexpr (FMT == DX_CACHE_I8) {
        constexpr float magic = 12582912.f;
        const uint32_t u = __float_as_uint(__fmaf_rn(a, inv, magic)), v = __float_as_uint(__fmaf_rn(b, inv, magic));
        const uint32_t w = __float_as_uint(__fmaf_rn(c, inv, magic)), x = __float_as_uint(__fmaf_rn(d, inv, magic));
        return __byte_perm(__byte_perm(u, v, 0x0040), __byte_perm(w, x, 0x0040), 0x5410);
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inv, d * inv), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}
// Two codes in the low half of `x` → two halfs (exact).
template <int FMT> __device__ __forceinline__ __half2 decode2(uint32_t x) {
    if constexpr (FMT == DX_CACHE_I8) {
        const uint32_t u = __byte_perm((x ^ 0x8080u), 0x64646464u, 0x4140);  // 1024 + (code + 128), twice
        return __hsub2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0x6480)));  // - 1152
    } else {
        uint32_t r;
        asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(x));
        return *reinterpret_cast<const __half2 *>(&r);
    }
}
// Four codes → four halfs, as the pairs (0,1) and (2,3) of the word.  FINITE: the codes 0x7F and 0xFF of e4m3, which no cache written
// here holds, come out as 448, so that what lies behind a mask (a weight of zero) cannot reach a result as a NaN.
template <int FMT, bool FINITE> __device__ __forceinline__ void decode4(uint32_t x, uint32_t &lo, uint32_t &hi) {
    if constexpr (FMT == DX_CACHE_I8) {
        x ^= 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half(0x6480));
        lo = __byte_perm(x, 0x64646464u, 0x4140);
        hi = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 a = __hsub2(*reinterpret_cast<const __half2 *>(&lo), off), b = __hsub2(*reinterpret_cast<const __half2 *>(&hi), off);
        lo = *reinterpret_cast<const uint32_t *>(&a);
        hi = *reinterpret_cast<const uint32_t *>(&b);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(x));
        if constexpr (FINITE) {
            const __half2 top = __half2half2(__ushort_as_half(0x5F00));
            const __half2 a = __hmin2(*reinterpret_cast<const __half2 *>(&lo), top), b = __hmin2(*reinterpret_cast<const __half2 *>(&hi), top);
            lo = *reinterpret_cast<const uint32_t *>(&a);
            hi = *reinterpret_cast<const uint32_t *>(&b);
        }
    }
}
#endif

}  // namespace kv
}  // namespace dx
