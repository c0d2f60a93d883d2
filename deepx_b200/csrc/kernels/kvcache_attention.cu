// dx_kvcache_attention: attention of packed new tokens over an 8-bit paged cache.
//
//   out[t,h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q[t,h].k_j - m),   c = scale log2(e),   j <= pos(t), j > pos(t) - window
//
// The rows of one sequence that share a key head (new token i, head i's group: n * group rows) are taken eight or sixteen at a time.
// For one new token a sequence this is bound by memory: every code is read once and used for a few rows.  Keys and values are the
// tensor cores' 16-row operand (sixteen tokens times a few rows; sixteen dimensions times a few rows), so that a group of up to eight
// rows wastes nothing and the halfs made of a code serve all rows at once.  One pass with the running maximum m and sum of the
// softmax; codes become halfs exactly, so the only rounding to 16 bits is that of the weights times their page's scale (and each row of a
// bfloat16 query is brought to size 1 by a power of two first, which keeps its 8 bits; elements 2^-17 below the row's largest begin to lose some).
//
// Work is split over the keys: the 64-token steps of all tiles of rows and heads of all sequences stand in one line, and each
// block takes an equal piece of it, whatever the lengths are (they are known on the device alone).  A piece may begin or end
// inside an item (one tile of rows, one head); such items' parts meet in the workspace and a second kernel joins them, always
// in the order of the keys: the same bits every time.
//
// Measured (B200, 32 query and 8 key heads of 128): one token after 262100, int8, f16: 94 to 101 us, 5.3 to 5.7 TB/s of the copy's 6.5; 64 single
// tokens after 300 to 8192, e4m3, bf16: 71 us, 4.7 TB/s, 7 of them the join; one token after 1500: 11 us on the device, two launches and
// the chain from the lengths to the pages to the keys; a prompt of 4096, 8 and 4 heads of 256: 930 us, as its keys are read and turned into halfs again for each
// sixteen rows.  More than the copy's time goes into each block's way to its first keys, the
// joints between items and turning codes into halfs with twelve warps an SM.
#include "kvcache_attention.cuh"

namespace dx {
namespace kv {
namespace {

constexpr int WARPS = 4, CTA = WARPS * 32;
constexpr int MIN_TOKENS = 128;  // of a block: fewer would cost more in joining than they save

// DP: the head's dimensions, padded; NB: blocks of eight rows of an item; WT: tokens a warp takes at a time, of one page.  What a turn of
// the loop costs besides its tokens (addresses, the wait, the vote on the maximum) is half of it at 16 tokens, so 32 are taken where the
// pages and the registers allow it (one token after 262100: 110 us with 16, 102 us with 32, on one card).
template <int DP, int NB, int WT> struct Cfg {
    static constexpr int ROWS = 8 * NB, STEP = WARPS * WT;
    static constexpr int STAGES = WT == 32 ? (DP == 64 ? 3 : 2) : DP == 64 ? 4 : 3;
    static constexpr int BLOCKS = DP == 256 ? 2 : NB == 1 && WT == 16 ? 4 : 3;  // resident on an SM
    static constexpr int TILE = WT * DP;                                            // bytes of a warp's keys (or values) of a stage
    static constexpr int RING = STAGES * 2 * TILE;                                  // of a warp; holds its ROWS x DP floats at the end
    static constexpr int SMEM = WARPS * RING;
    static constexpr int PART = ROWS * DP + 2 * ROWS;  // floats of a part in the workspace: output, m, l
    static_assert(RING >= ROWS * DP * 4, "the ring holds a warp's output");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of halfs: lane (g, t) gives row g, columns 2t and 2t+1 and takes column g, rows 2t and 2t+1.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Where chunk `c` (16 bytes) of token `r` of a warp's tile lies: rows of DP bytes whose chunks are exchanged so that both ways the
// tile is read (eight tokens, every other chunk; four tokens of one parity, two chunks) touch every bank once.
template <int DP> __device__ __forceinline__ int place(int r, int c) {
    if constexpr (DP == 64) return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ ((r >> 1) & 7)) << 4);
    else return r * DP + ((c ^ (r & 7)) << 4);
}
// The chunk that lane t of a quad multiplies in its i-th turn.
template <int DP> __device__ __forceinline__ int key_chunk(int t, int i) { return DP == 64 ? t : 2 * t + (i & 1) + 8 * (i >> 1); }

// One sequence as the line of steps sees it.
struct Line {
    int lo, steps, tiles;  // first token of the range (a multiple of STEP), steps of a tile of rows, tiles of rows of a head
};
template <int ROWS, int STEP> __device__ __forceinline__ Line line_of(const Seq &q, const Attn &a) {
    Line l;
    const int64_t hi = min(int64_t(q.end), int64_t(q.first) + q.n);
    const int64_t lo = a.window > 0 ? max(int64_t(0), int64_t(q.first) - a.window + 1) : 0;
    l.lo = int(min(lo, max(hi, int64_t(0))) / STEP * STEP);
    l.steps = hi > l.lo ? int((hi - l.lo + STEP - 1) / STEP) : 1;  // a row that sees nothing is written too
    l.tiles = int((int64_t(q.n) * a.group + ROWS - 1) / ROWS);
    return l;
}
template <int ROWS, int STEP> __device__ __forceinline__ int64_t steps_of(const Seqs &s, const Cache &c, const Attn &a, int b) {
    const Seq q = seq_at(s, c, b);
    if (q.n == 0) return 0;
    const Line l = line_of<ROWS, STEP>(q, a);
    return int64_t(l.steps) * l.tiles * c.heads;
}

template <typename T, int FMT, int DP, int NB, int WT>
__global__ void __launch_bounds__(CTA, Cfg<DP, NB, WT>::BLOCKS) attention_kernel(Attn a, Cache c, Seqs s) {
    using K = Cfg<DP, NB, WT>;
    constexpr int ROWS = K::ROWS, STEP = K::STEP, TT = WT / 16;  // TT: tiles of sixteen tokens
    constexpr int MT = DP / 16;            // tiles of sixteen dimensions of the output
    constexpr int KC = DP / 64;            // chunks of a key that a lane multiplies
    constexpr int VC = DP == 256 ? 2 : 1;  // chunks of a value that a lane multiplies (half of one at DP 64)
    extern __shared__ __align__(1024) uint8_t ring[];
    __shared__ float scales[WARPS][K::STAGES][2];
    __shared__ int in_cache[WARPS][K::STAGES];
    __shared__ float sm_m[WARPS][ROWS], sm_l[WARPS][ROWS];
    __shared__ int64_t before[CTA], total_steps;
    __shared__ int64_t found_at;
    __shared__ int found_b;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    griddep_wait_cta();
    if (blockIdx.x == gridDim.x - 1) check_seqs(s, c, a.flag);  // a block that has no piece when there is little to do

    // ---- this block's piece of the line ----
    const int per = (s.batch + CTA - 1) / CTA;
    {
        int64_t mine = 0;
        for (int b = threadIdx.x * per; b < min(s.batch, int(threadIdx.x + 1) * per); ++b) mine += steps_of<ROWS, STEP>(s, c, a, b);
        int64_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        if (lane == 31) before[warp] = sum;
        __syncthreads();
        int64_t base = 0;
        for (int w = 0; w < warp; ++w) base += before[w];
        __syncthreads();
        before[threadIdx.x] = base + sum - mine;
        if (threadIdx.x == CTA - 1) total_steps = base + sum;
        __syncthreads();
    }
    const int64_t total = total_steps;
    const int64_t blocks = max(int64_t(1), min(int64_t(gridDim.x), total * STEP / MIN_TOKENS));
    Join *join = reinterpret_cast<Join *>(a.ws) + blockIdx.x;
    float *parts = reinterpret_cast<float *>(a.ws + gridDim.x * sizeof(Join));
    if (total == 0 || int64_t(blockIdx.x) >= blocks) {
        if (threadIdx.x == 0) join->parts = 0;
        return;
    }
    const int64_t begin = total * blockIdx.x / blocks, end = total * (blockIdx.x + 1) / blocks;
    if (before[threadIdx.x] <= begin && (threadIdx.x == CTA - 1 || before[threadIdx.x + 1] > begin)) {
        int64_t at = before[threadIdx.x];
        int b = threadIdx.x * per;
        for (; b < s.batch; ++b) {
            const int64_t n = steps_of<ROWS, STEP>(s, c, a, b);
            if (at + n > begin) break;
            at += n;
        }
        found_b = b;
        found_at = at;
    }
    __syncthreads();
    int b = found_b;
    int64_t seq_begin = found_at;
    if (threadIdx.x == 0) join->parts = 0;

    uint8_t *my_ring = ring + warp * K::RING;
    const uint32_t ring_u = smem_u32(my_ring);
    // the sixteen bytes of a tile that this lane loads first; the others lie whole rows further
    const int lane_row = lane / (DP / 16), lane_chunk = lane % (DP / 16), lane_src = lane_row * c.dim + lane_chunk * 16, row_step = (512 / DP) * c.dim;
    const bool lane_in = lane_chunk * 16 < c.dim;
    // where this lane's parts of a tile lie in a stage: to load (rows of either parity of 512 / DP), keys, values of even and odd tokens
    const uint32_t load_at = place<DP>(lane_row, lane_chunk), load_odd = load_at ^ 64;
    const uint32_t key_at = place<DP>(g, key_chunk<DP>(t, 0));
    const int value_half = DP == 64 ? (g & 1) * 8 : 0;
    const uint32_t value_at = place<DP>(2 * t, DP == 64 ? g >> 1 : g) + value_half, value_odd = place<DP>(2 * t + 1, DP == 64 ? g >> 1 : g) + value_half;
    auto later = [](uint32_t at) { return (DP == 64 ? at ^ 64 : at) + 8 * DP; };  // the same of the token eight further
    const int64_t page_bytes = int64_t(c.heads) * c.page * c.dim;
    for (int64_t at = begin; at < end;) {
        const Seq sq = seq_at(s, c, b);
        const Line ln = line_of<ROWS, STEP>(sq, a);
        const int64_t seq_steps = sq.n ? int64_t(ln.steps) * ln.tiles * c.heads : 0;
        if (at >= seq_begin + seq_steps) {  // on to the next sequence
            seq_begin += seq_steps;
            ++b;
            continue;
        }
        const int64_t item = (at - seq_begin) / ln.steps;
        const int64_t item_begin = seq_begin + item * ln.steps, item_end = item_begin + ln.steps;
        const int step0 = int(at - item_begin), step1 = int(min(end, item_end) - item_begin);
        const int head = int(item / ln.tiles), first_row = int(item - int64_t(head) * ln.tiles) * ROWS;
        const int rows = min(ROWS, int(min(int64_t(sq.n) * a.group - first_row, int64_t(ROWS))));
        const int steps = step1 - step0;

        const int pos_min = sq.first + first_row / a.group, pos_max = sq.first + (first_row + rows - 1) / a.group;
        const int seen_end = min(sq.end, pos_max + 1);  // tokens from here on are no row's, and those in front of seen_begin: their pages may be anyone's
        const int seen_begin = a.window > 0 ? int(max(int64_t(pos_min) - a.window + 1, int64_t(0))) : 0;

        float o[NB][MT][4], l[NB][2];  // output, sum (of this lane's tokens)
        Maxima most[NB][2];
        float unit[NB][2];  // 2^(7 - d)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            most[nb][0].clear();
            most[nb][1].clear();
            unit[nb][0] = unit[nb][1] = exp2_approx(UP - D_LEAST);
            l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < MT; ++d) o[nb][d][e] = 0.f;
        }

        // ---- keys and values in flight ----
        const int32_t *table = s.table + int64_t(b) * s.cols;
        const int64_t head_bytes = int64_t(head) * c.page * c.dim;
        auto token0 = [&](int step) { return ln.lo + (step0 + step) * STEP + warp * WT; };
        auto page_number = [&](int step) {
            const int j = token0(step);
            return step < steps && j < seen_end && j + WT > seen_begin ? table[j >> c.page_shift] : -1;
        };
        auto issue = [&](int step, int stage, int32_t number) {
            if (step < steps) {
                const int j = token0(step);
                const int left = j + WT > seen_begin ? seen_end - j : 0;  // tokens to load
                const bool ok = left > 0 && number >= 0 && number < c.pages;
                if (left > 0 && !ok && lane == 0) raise(a.flag, FLAG_PAGE);
                const uint32_t dst = ring_u + stage * 2 * K::TILE;
                const int64_t base = ok ? number * page_bytes + head_bytes + (j & (c.page - 1)) * c.dim : 0;
                const uint8_t *ksrc = c.k + (base + lane_src), *vsrc = c.v + (base + lane_src);
                if (ok && left >= WT && c.dim == DP) {
#pragma unroll
                    for (int i = 0; i < K::TILE / 512; ++i) {
                        const uint32_t at = dst + (DP == 256 ? place<DP>(i * 2 + lane_row, lane_chunk) : (i & 1 ? load_odd : load_at) + i * 512);
                        cp_async16(at, ksrc + i * 512, true);
                        cp_async16(at + K::TILE, vsrc + i * 512, true);
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < K::TILE / 512; ++i) {
                        const bool in = ok && lane_in && i * (512 / DP) + lane_row < left;
                        const uint32_t at = dst + place<DP>(i * (512 / DP) + lane_row, lane_chunk);
                        const int64_t off = in ? int64_t(i) * row_step : 0;
                        cp_async16(at, in ? ksrc + off : c.k, in);
                        cp_async16(at + K::TILE, in ? vsrc + off : c.v, in);
                    }
                }
                const int64_t ph = ok ? int64_t(number) * c.heads + head : 0;
                if (lane < 2) cp_async4(smem_u32(&scales[warp][stage][lane]), (lane ? c.v_scale : c.k_scale) + ph, ok);
                if (lane == 2) in_cache[warp][stage] = ok;
            }
            cp_commit();
        };
        int32_t next = page_number(0);
#pragma unroll
        for (int p = 0; p < K::STAGES - 1; ++p) {
            const int32_t number = next;
            next = page_number(p + 1);
            issue(p, p, number);
        }

        // ---- the queries, while the first keys are on their way: row g of each block of eight, the chunks this lane multiplies ----
        uint32_t qb[NB][KC][4][2];
        float c_row[NB][2];  // of the rows 2t and 2t + 1, whose scores this lane has
        int pos[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int r = 8 * nb + g, fr = first_row + r;
            const bool live = r < rows;
            const int i = live ? fr / a.group : 0;
            const T *q = static_cast<const T *>(a.q) + (sq.row0 + i) * a.q_stride + int64_t(head * a.group + (live ? fr - i * a.group : 0)) * c.dim;
            Pack<T, 8> x[KC][2];
            float amax = 0.f;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                const int d = key_chunk<DP>(t, k) * 16;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (live && d < c.dim && a.q_vec) x[k][h] = ld_cached<T, 8>(q + d + 8 * h);
                    else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[k][h].v[e] = live && d < c.dim ? q[d + 8 * h + e] : from_compute<T>(0.f);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(to_compute(x[k][h].v[e])));
                }
            }
            float down = 1.f, c_mine = a.scale_log2;
            if constexpr (std::is_same<T, bf16>::value) {
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const uint32_t e = min(max(__float_as_uint(amax) >> 23, 1u), 253u);
                if (amax > 0.f && amax < __int_as_float(0x7f800000)) {
                    down = __uint_as_float((254u - e) << 23);
                    c_mine *= __uint_as_float(e << 23);
                }
            }
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int w = 0; w < 4; ++w) {  // word w of the chunk: dimensions 4w..4w+3
                    const Pack<T, 8> &p = x[k][w >> 1];
                    const int e = (w & 1) * 4;
                    qb[nb][k][w][0] = half2_bits(to_compute(p.v[e]) * down, to_compute(p.v[e + 1]) * down);
                    qb[nb][k][w][1] = half2_bits(to_compute(p.v[e + 2]) * down, to_compute(p.v[e + 3]) * down);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = 8 * nb + 2 * t + e;
                c_row[nb][e] = __shfl_sync(0xffffffffu, c_mine, (2 * t + e) * 4);
                pos[nb][e] = col < rows ? sq.first + (first_row + col) / a.group : INT32_MIN;
            }
        }
        int stage = 0;
        for (int step = 0; step < steps; ++step) {
            cp_wait<K::STAGES - 2>();
            __syncwarp();  // the stage has arrived, and every lane is done with the one before it
            {
                const int32_t number = next;
                next = page_number(step + K::STAGES);
                issue(step + K::STAGES - 1, stage == 0 ? K::STAGES - 1 : stage - 1, number);
            }
            const uint32_t ks = ring_u + stage * 2 * K::TILE, vs = ks + K::TILE;
            const float k_scale = scales[warp][stage][0], v_scale = scales[warp][stage][1];
            const bool ok = in_cache[warp][stage];
            const int j0 = token0(step);
            if (++stage == K::STAGES) stage = 0;
            if (!ok) continue;  // no token of a page: nothing to see

            // ---- scores: lane (g, t) holds tokens g, g+8 (of each sixteen) of rows 2t, 2t+1 ----
            float x[NB][TT][4];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[nb][tt][e] = 0.f;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                // the second chunk is the first one's neighbour, the third and fourth lie 128 bytes further
                const uint32_t at = (key_at ^ ((k & 1) << 4)) + (k >> 1) * 128;
                uint4 w0[TT], w1[TT];
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    w0[tt] = lds128(ks + at + tt * 16 * DP);
                    w1[tt] = lds128(ks + later(at) + tt * 16 * DP);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) {
                        const uint32_t lo[4] = {w0[tt].x, w0[tt].y, w0[tt].z, w0[tt].w}, hi[4] = {w1[tt].x, w1[tt].y, w1[tt].z, w1[tt].w};
                        uint32_t ka[4];
                        decode4<FMT, false>(lo[i], ka[0], ka[2]);
                        decode4<FMT, false>(hi[i], ka[1], ka[3]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) mma(x[nb][tt], ka, qb[nb][k][i][0], qb[nb][k][i][1]);
                    }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float c0 = c_row[nb][0] * k_scale, c1 = c_row[nb][1] * k_scale;
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[nb][tt][e] *= e & 1 ? c1 : c0;
            }
            const bool masked = j0 + WT - 1 > pos_min || j0 + WT > sq.end || (a.window > 0 && j0 <= int64_t(pos_max) - a.window);
            if (masked) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = j0 + 16 * tt + g + 8 * (e >> 1), p = pos[nb][e & 1];
                            const bool seen = j <= p && j < sq.end && (a.window <= 0 || j > int64_t(p) - a.window);
                            if (!seen) x[nb][tt][e] = NEG_INF;
                        }
            }
            // ---- running maxima: a row's rise when a score is 2^8 above one of them ----
            const float power = scale_power(v_scale);
            float top[NB][2];
            bool rise = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v = fmaxf(x[nb][0][e], x[nb][0][e + 2]);
#pragma unroll
                    for (int tt = 1; tt < TT; ++tt) v = fmaxf(v, fmaxf(x[nb][tt][e], x[nb][tt][e + 2]));
                    rise |= v - most[nb][e].m > fminf(LAG, most[nb][e].d + (LAG - power));
                    top[nb][e] = v;
                }
            if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float by[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = top[nb][e], of_sum;
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
                        most[nb][e].rise(v, [&](float m) { return v - m + power; }, of_sum, by[e]);
                        l[nb][e] *= of_sum;
                        unit[nb][e] = exp2_approx(UP - most[nb][e].d);
                    }
#pragma unroll
                    for (int d = 0; d < MT; ++d) {
                        o[nb][d][0] *= by[0];
                        o[nb][d][1] *= by[1];
                        o[nb][d][2] *= by[0];
                        o[nb][d][3] *= by[1];
                    }
                }
            }
            uint32_t p[NB][TT][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                // finite also for a row that does not see the page
                const float h0 = fminf(unit[nb][0] * v_scale, -LOWEST), h1 = fminf(unit[nb][1] * v_scale, -LOWEST), m0 = most[nb][0].m, m1 = most[nb][1].m;
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    const float y0 = exp2_approx(x[nb][tt][0] - m0), y1 = exp2_approx(x[nb][tt][1] - m1), y2 = exp2_approx(x[nb][tt][2] - m0), y3 = exp2_approx(x[nb][tt][3] - m1);
                    l[nb][0] += y0 + y2;
                    l[nb][1] += y1 + y3;
                    p[nb][tt][0] = transpose8(half2_bits(y0 * h0, y1 * h1));
                    p[nb][tt][1] = transpose8(half2_bits(y2 * h0, y3 * h1));
                }
            }

            // ---- values: lane (g, t) multiplies tokens 2t, 2t+1, 2t+8, 2t+9 of its chunk's dimensions ----
            // FINITE: some of the tile's tokens are masked for some rows; what lies there must not be no number.
            auto values = [&](auto finite) {
                auto four = [&](int tt, uint32_t wa, uint32_t wb, uint32_t wc, uint32_t wd, int tile) {
                    uint32_t v0[4], v1[4];  // of dimensions 2 tile, 2 tile + 1 and the two after: tokens 2t.., tokens 2t + 8..
                    decode4<FMT, decltype(finite)::value>(__byte_perm(wa, wb, 0x5140), v0[0], v0[1]);
                    decode4<FMT, decltype(finite)::value>(__byte_perm(wc, wd, 0x5140), v0[2], v0[3]);
                    decode4<FMT, decltype(finite)::value>(__byte_perm(wa, wb, 0x7362), v1[0], v1[1]);
                    decode4<FMT, decltype(finite)::value>(__byte_perm(wc, wd, 0x7362), v1[2], v1[3]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        mma(o[nb][tile], v0, p[nb][tt][0], p[nb][tt][1]);
                        mma(o[nb][tile + 1], v1, p[nb][tt][0], p[nb][tt][1]);
                    }
                };
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    const uint32_t even = vs + tt * 16 * DP + value_at, odd = vs + tt * 16 * DP + value_odd;
                    const uint32_t even8 = vs + tt * 16 * DP + later(value_at), odd8 = vs + tt * 16 * DP + later(value_odd);
                    if constexpr (DP == 64) {
                        const uint2 wa = lds64(even), wb = lds64(odd), wc = lds64(even8), wd = lds64(odd8);
                        four(tt, wa.x, wb.x, wc.x, wd.x, 0);
                        four(tt, wa.y, wb.y, wc.y, wd.y, 2);
                    } else {
#pragma unroll
                        for (int h = 0; h < VC; ++h) {
                            const uint4 wa = lds128(even + 128 * h), wb = lds128(odd + 128 * h), wc = lds128(even8 + 128 * h), wd = lds128(odd8 + 128 * h);
                            four(tt, wa.x, wb.x, wc.x, wd.x, 8 * h);
                            four(tt, wa.y, wb.y, wc.y, wd.y, 8 * h + 2);
                            four(tt, wa.z, wb.z, wc.z, wd.z, 8 * h + 4);
                            four(tt, wa.w, wb.w, wc.w, wd.w, 8 * h + 6);
                        }
                    }
                }
            };
            if (FMT == DX_CACHE_E4M3 && masked) values(std::true_type());
            else values(std::false_type());
        }
        cp_wait<0>();
        __syncthreads();  // every warp is done with its ring

        // ---- the four warps' parts, each divided by its own sum, into the rings ----
        constexpr int W = DP == 64 ? 8 : 16;  // dimensions of a lane's run
        auto in_part = [&](int row, int d) { return row * DP + (((d >> 2) ^ ((row >> 1) & 3)) << 2); };
        float *mine = reinterpret_cast<float *>(my_ring);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[nb][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const Out by = way_out(most[nb][e].d, sum);
                auto result = [&](float x) { return x * by.first * by.second; };
                const int row = 8 * nb + 2 * t + e;
                if (g == 0) {
                    sm_m[warp][row] = most[nb][e].m;
                    sm_l[warp][row] = sum;
                }
#pragma unroll
                for (int h = 0; h < VC; ++h)
#pragma unroll
                    for (int i = 0; i < W; i += 4) {
                        const int d = h * 128 + g * W + i, tile = h * 8 + i / 2;
                        *reinterpret_cast<float4 *>(mine + in_part(row, d)) =
                            make_float4(result(o[nb][tile][e]), result(o[nb][tile][2 + e]), result(o[nb][tile + 1][e]), result(o[nb][tile + 1][2 + e]));
                    }
            }
        __syncthreads();
        const bool whole = step0 == 0 && step1 == ln.steps;
        float *part = parts + (int64_t(blockIdx.x) * 2 + (step0 == 0 ? 1 : 0)) * K::PART;
        for (int u = threadIdx.x; u < ROWS * (DP / 4); u += CTA) {
            const int row = u / (DP / 4), d = (u - row * (DP / 4)) * 4;
            if (row >= rows || d >= c.dim) continue;
            float top = NEG_INF, sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_m[w][row]);
            const float base = or_zero(top);
            float share[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum += share[w] = sm_l[w][row] * exp2_approx(sm_m[w][row] - base);
            const float all = sum == 0.f ? 0.f : 1.f / sum;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float by = share[w] * all;  // shares of one: a sum that is divided afterwards could be out of range
                const float4 x = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(ring + w * K::RING) + in_part(row, d));
                v.x += by * x.x;
                v.y += by * x.y;
                v.z += by * x.z;
                v.w += by * x.w;
            }
            if (whole) {
                const int fr = first_row + row, i = fr / a.group;
                T *out = static_cast<T *>(a.out) + (sq.row0 + i) * a.out_stride + int64_t(head * a.group + fr - i * a.group) * c.dim + d;
                Pack<T, 4> y;
                y.v[0] = from_compute<T>(v.x);
                y.v[1] = from_compute<T>(v.y);
                y.v[2] = from_compute<T>(v.z);
                y.v[3] = from_compute<T>(v.w);
                if (a.out_vec) st_stream<T, 4>(out, y);
                else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[e] = y.v[e];
                }
            } else {
                *reinterpret_cast<float4 *>(part + row * DP + d) = v;
                if (d == 0) {
                    part[ROWS * DP + row] = top;
                    part[ROWS * DP + ROWS + row] = sum;
                }
            }
        }
        // the item begins in the block before and this block's begin lies inside it: here is where it is joined
        if (threadIdx.x == 0 && at == begin && step0 > 0 && item_begin >= total * (int64_t(blockIdx.x) - 1) / blocks) {
            join->row0 = sq.row0;
            join->first_row = first_row;
            join->rows = rows;
            join->head = head;
            join->parts = int((item_end * blocks - 1) / total) - int(blockIdx.x) + 2;  // the last block that has steps of it
        }
        __syncthreads();  // the rings are free again
        at = item_begin + step1;
    }
}

template <typename T, int FMT, int DP, int NB, int WT> int launch_tokens(const Attn &a, const Cache &c, const Seqs &s, cudaStream_t st) {
    using K = Cfg<DP, NB, WT>;
    static std::atomic<uint64_t> prepared{0};  // one bit for each device
    if (int e = allow_shared(attention_kernel<T, FMT, DP, NB, WT>, K::SMEM, &prepared)) return e;
    const unsigned grid = unsigned(sm_count() * K::BLOCKS);
    launch_pdl(attention_kernel<T, FMT, DP, NB, WT>, dim3(grid), dim3(CTA), K::SMEM, st, a, c, s);
    if (int e = check_launch("kvcache_attention")) return e;
    launch_pdl(join_kernel<T, DP, K::ROWS>, dim3(grid), dim3(JOIN_CTA), 0, st, a, c);
    return check_launch("kvcache_attention (join)");
}
// Up to eight rows of up to 128 dimensions leave registers for 32 tokens at a time; pages of sixteen hold no 32.
template <typename T, int FMT, int DP> int launch(const Attn &a, const Cache &c, const Seqs &s, int64_t rows, cudaStream_t st) {
    if (rows > 8) return launch_tokens<T, FMT, DP, 2, 16>(a, c, s, st);
    if constexpr (DP <= 128)
        if (c.page >= 32) return launch_tokens<T, FMT, DP, 1, 32>(a, c, s, st);
    return launch_tokens<T, FMT, DP, 1, 16>(a, c, s, st);
}

// Large enough for every variant of the head's dimensions.
template <int DP> size_t workspace_of() {
    const size_t one = Cfg<DP, 1, 16>::BLOCKS * (sizeof(Join) + 2 * Cfg<DP, 1, 16>::PART * sizeof(float));
    const size_t two = Cfg<DP, 2, 16>::BLOCKS * (sizeof(Join) + 2 * Cfg<DP, 2, 16>::PART * sizeof(float));
    return size_t(sm_count()) * (one > two ? one : two);
}
int padded(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
size_t workspace(int dim) { return dim <= 64 ? workspace_of<64>() : dim <= 128 ? workspace_of<128>() : workspace_of<256>(); }
// Whether a call goes to the tiles of 128 rows, whose time hardly depends on the rows: here every sixteen rows of a sequence and key head
// read its cache again.  64 sequences of 4096 tokens, 8 key heads, here against the tiles: 32 rows of 128 dimensions 265 us against 385,
// 48 rows 387 against 387, 64 rows 506 against 390; of 64 dimensions 64 rows 337 against 369, 96 rows 502 against 371.  (Eight
// sequences: 48 rows of 128 dimensions 62 against 51 us, 64 rows of 64 52 against 48.)
bool by_tiles(const Cache &c, int64_t rows) { return c.dim <= 128 && rows > (c.dim <= 64 ? 64 : 32); }
// The most rows of a sequence that share a key head, as far as the caller says.
int64_t rows_of(int64_t q_heads, const Cache &c, const Seqs &s, int64_t max_new) {
    return (max_new > 0 && max_new < s.rows ? max_new : s.rows) * (q_heads / c.heads);
}

}  // namespace
}  // namespace kv
}  // namespace dx

extern "C" size_t dx_kvcache_attention_workspace_bytes(int dtype, int64_t q_heads, const dx_kvseqs *seqs, const dx_kvcache *cache, int64_t max_new) {
    using namespace dx;
    kv::Cache c;
    kv::Seqs s;
    if (kv::check("kvcache_attention", cache, seqs, &c, &s) || s.rows == 0 || s.batch == 0) return 0;
    if (q_heads < 1 || q_heads % c.heads) return 0;
    const int64_t rows = kv::rows_of(q_heads, c, s, max_new);
    return kv::by_tiles(c, rows) ? kv::tiles_workspace(c, s, int(q_heads / c.heads)) : kv::workspace(c.dim);
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
    if (!(scale > 0) || !(float(scale * 1.4426950408889634) > 0) || scale > 1e38) return fail(DX_E_ARG, "kvcache_attention: scale %g", scale);
    if (max_new < 0 || window < 0) return fail(DX_E_ARG, "kvcache_attention: max_new %lld, window %lld", (long long)max_new, (long long)window);
    if (s.rows * (q_heads / c.heads) > INT32_MAX) return fail(DX_E_SHAPE, "kvcache_attention: %lld rows of %lld heads each over a key head", (long long)s.rows, (long long)(q_heads / c.heads));
    if (s.rows == 0 || s.batch == 0) return DX_OK;
    if (!q || !out) return fail(DX_E_ARG, "kvcache_attention: null tensor pointer");
    const Span qs = span(q, s.rows, q_stride * 2, width * 2), outs = span(out, s.rows, out_stride * 2, width * 2), raised = span(flag, 4);
    const kv::CacheSpans spans(c, s);
    if (meet(outs, qs) || spans.met_by(outs)) return fail(DX_E_ALIAS, "kvcache_attention: the output overlaps an input");
    if (meet(outs, raised) || meet(qs, raised) || spans.met_by(raised)) return fail(DX_E_ALIAS, "kvcache_attention: the flag lies in a tensor");
    const int64_t rows = kv::rows_of(q_heads, c, s, max_new);
    const bool tiles = kv::by_tiles(c, rows);
    const size_t need = tiles ? kv::tiles_workspace(c, s, int(q_heads / c.heads)) : kv::workspace(c.dim);
    if (!workspace || workspace_bytes < need) return fail(DX_E_WORKSPACE, "kvcache_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (!aligned_to(workspace, 256)) return fail(DX_E_ARG, "kvcache_attention: the workspace must start on a 256-byte boundary");
    const Span scratch = span(workspace, int64_t(need));
    if (meet(scratch, outs) || meet(scratch, qs) || meet(scratch, raised) || spans.met_by(scratch)) return fail(DX_E_ALIAS, "kvcache_attention: the workspace overlaps a tensor");
    kv::Attn a{q, out, q_stride, out_stride, int(q_heads), int(q_heads / c.heads), int(window > INT32_MAX ? 0 : window), float(scale * 1.4426950408889634),
               q_stride % 8 == 0 && aligned_to(q, 16), out_stride % 8 == 0 && aligned_to(out, 16), static_cast<uint8_t *>(workspace), flag};
    cudaStream_t st = as_stream(stream);
    if (tiles) return kv::launch_tiles(dtype, cache->format, a, c, s, st);
#define DX_CALL(T, FMT)                                                             \
    switch (kv::padded(c.dim)) {                                                    \
        case 64: return kv::launch<T, FMT, 64>(a, c, s, rows, st);                        \
        case 128: return kv::launch<T, FMT, 128>(a, c, s, rows, st);                      \
        default: return kv::launch<T, FMT, 256>(a, c, s, rows, st);                       \
    }
    if (dtype == DX_F16) {
        if (cache->format == DX_CACHE_I8) { DX_CALL(f16, DX_CACHE_I8) }
        DX_CALL(f16, DX_CACHE_E4M3)
    }
    if (cache->format == DX_CACHE_I8) { DX_CALL(bf16, DX_CACHE_I8) }
    DX_CALL(bf16, DX_CACHE_E4M3)
#undef DX_CALL
}
