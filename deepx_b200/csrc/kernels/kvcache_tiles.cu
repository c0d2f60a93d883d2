// dx_kvcache_attention for prompts: tiles of 128 rows on tcgen05 tensor cores.
//
// An item is up to 256 rows (new token i, head of the key head's group: i * group + g, flattened) of one sequence and key head, two
// tiles of 128 rows.  For each step of 64 keys and each tile:
//     S = Q K^T          128 x 64, into one of the tile's two places in TMEM;  Q, K halfs in shared memory
//     P = 2^(c S - m)    a thread has a row; halfs, over S's place
//     O = O + P V        128 x dim, in TMEM, P from TMEM;                      V halfs in shared memory
// The scores are issued two steps ahead, so a tile's softmax finds the next ones ready when it is done with the last.  512 multiply-adds
// go with each exponential at 128 dimensions: 64 keys of both tiles cost 1024 cycles of the tensor cores and 1024 of the exponential
// unit, so both would bound a perfect kernel; what is neither stays off their threads.
//
// Roles (16 warps, one block an SM): warps 0-3 and 4-7 the softmax of a tile each; 8-10 turn the codes of K into halfs, 11-13 those of V
// (sixteen a thread and turn, loaded a step ahead); a thread of warp 14 and one of 15 issue a tile's products each.  Codes become halfs
// unscaled and exact; the scales of a step's groups of sixteen tokens go to the softmax threads, K's into the factor c, V's into
// the exponent, so they cost no instruction for each element.  A row's maximum may lag by 2^8 before O is
// scaled again (in TMEM, by the row's thread), which after the first steps hardly happens.
//
// Measured (B200): two prompts of 4096 tokens, 32 query and 8 key heads of 128, int8, bf16: 400 to 406 us with the plan and the join (14 us), 683 TFLOP/s,
// 0.42 of a large matrix product's rate, 242 us with a window of 1024; 12 sequences of 1 to 700 new tokens up to 5000, 14 and 2 heads of 64: 94 us.
// 2 to 4 % of it is what the values' scales cost in the maximum and the sum.  A step of 64 keys takes, without that, about 2800 cycles:
// 1300 the exponentials and weights of a row, 560 its maximum, 380 and 270 the waits before and after, while the first converter's way through a step is nearly as long (with the exponentials left out the kernel waits for keys and gains 4 %, with the
// conversion left out 2 %).  Not taken, as slower: two threads a row (16 softmax warps of 80 registers: 520 us), the tiles in turns, loading
// the next scores early, weights times their page's scale in place of a common exponent (windowed 246 us, two prompts with heads of 64 170 in place of 165).
//
// The steps of all items stand in one line, planned by a small kernel first, and every block takes an equal piece of it, where an
// item counts OVERHEAD steps more than it has (its queries, its way out: 13,000 to 15,000 cycles measured, five steps of 2800, counted as six for heads of either size; without that the blocks of a prompt's first
// rows, whose items have few steps, took twice the others' time); items that more than one block works on are joined as in kvcache_attention.cu.
//
// Every wait is bounded by a clock; when one runs out a status word is set (dx_kvcache_status), all roles leave, TMEM is freed.
#include <mutex>

#include "kvcache_attention.cuh"

namespace dx {
namespace kv {
namespace {

constexpr int TILE_ROWS = 128, ITEM_ROWS = 256, KEYS = 64, GROUPS = KEYS / 16;
constexpr int THREADS = 16 * 32;
// Info of a step outlives its keys: its place is written again when the scores of four steps later are complete, which were issued
// behind the weights of two steps later.
constexpr int STAGES = 4, INFO = 8;
constexpr int CONVERTERS = 3;  // warps for K, and for V
constexpr int OVERHEAD = 6;
constexpr int PLAN_CTA = 1024;
constexpr float CAP = 100.f, CAP_INVERSE = 0x1p100f;
constexpr long long WAIT_LIMIT_CYCLES = 4000000000ll;  // ~2 s
enum Status : int { S_OK = 0, S_KEYS = 1, S_VALUES = 2, S_SCORES = 3, S_WEIGHTS = 4, S_QUERIES = 5, S_OUTPUT = 6, S_ROOM = 7 };

__device__ int g_status = 0;

// 256 rows of a sequence, the same for all heads: rows first_row.. of the flattened (new token, head of the group), tokens lo..hi
// in steps of KEYS from lo (a multiple of KEYS); the first token that one of the rows sees (pages wholly in front of it may be anyone's).
struct alignas(16) Group {
    int64_t row0;
    int b, first, end;  // sequence, position of its first new token, tokens its pages can be read for
    int first_row, rows, lo, hi, steps, first_seen;
};
// The plan: the groups, the units of the line in front of each, the groups in front of a sequence.
struct Plan {
    int64_t *before;  // [groups + 1]
    Group *group;
    int *first;  // [batch + 1]
    int *count;  // groups
};
__host__ __device__ inline int64_t most_groups(const Seqs &s, int group) { return s.rows * group / ITEM_ROWS + s.batch; }
__host__ __device__ inline size_t align256(size_t n) { return (n + 255) & ~size_t(255); }
__host__ __device__ inline Plan plan_at(uint8_t *base, const Seqs &s, int group) {
    const int64_t n = most_groups(s, group);
    Plan p;
    p.before = reinterpret_cast<int64_t *>(base);
    base += align256(size_t(n + 1) * 8);
    p.group = reinterpret_cast<Group *>(base);
    base += align256(size_t(n) * sizeof(Group));
    p.first = reinterpret_cast<int *>(base);
    base += align256(size_t(s.batch + 1) * 4);
    p.count = reinterpret_cast<int *>(base);
    return p;
}
inline size_t plan_bytes(const Seqs &s, int group) {
    const int64_t n = most_groups(s, group);
    return align256(size_t(n + 1) * 8) + align256(size_t(n) * sizeof(Group)) + align256(size_t(s.batch + 1) * 4) + 256;
}

__device__ __forceinline__ Group group_of(const Seq &q, const Attn &a, int b, int tile) {
    Group x;
    x.row0 = q.row0;
    x.b = b;
    x.first = q.first;
    x.end = q.end;
    x.first_row = tile * ITEM_ROWS;
    x.rows = int(min(int64_t(q.n) * a.group - x.first_row, int64_t(ITEM_ROWS)));
    const int64_t p0 = int64_t(q.first) + x.first_row / a.group, p1 = int64_t(q.first) + (x.first_row + x.rows - 1) / a.group;
    const int64_t hi = max(min(int64_t(q.end), p1 + 1), int64_t(0));
    const int64_t lo = a.window > 0 ? max(int64_t(0), p0 - a.window + 1) : 0;
    x.hi = int(hi);
    x.first_seen = int(min(lo, hi));
    x.lo = x.first_seen / KEYS * KEYS;
    x.steps = hi > x.lo ? int((hi - x.lo + KEYS - 1) / KEYS) : 1;  // rows that see nothing are written too
    return x;
}

__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sum, int64_t &total) {  // exclusive, PLAN_CTA threads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += up;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int64_t base = 0, all = 0;
    for (int w = 0; w < PLAN_CTA / 32; ++w) {
        if (w < warp) base += warp_sum[w];
        all += warp_sum[w];
    }
    total = all;
    return base + s - v;
}

__global__ void __launch_bounds__(PLAN_CTA) plan_kernel(Attn a, Cache c, Seqs s, Plan p) {
    __shared__ int64_t warp_sum[PLAN_CTA / 32];
    griddep_wait_cta();
    check_seqs(s, c, a.flag);
    const int64_t room = most_groups(s, a.group);
    int64_t groups = 0;
    for (int b0 = 0; b0 < s.batch; b0 += PLAN_CTA) {
        const int b = b0 + threadIdx.x;
        int64_t n = 0, total;
        if (b < s.batch) n = (int64_t(seq_at(s, c, b).n) * a.group + ITEM_ROWS - 1) / ITEM_ROWS;
        const int64_t at = groups + block_scan(n, warp_sum, total);
        if (b < s.batch) p.first[b] = int(min(at, room));
        groups += total;
    }
    groups = min(groups, room);  // starts that overlap could ask for more than the rows allow; check_seqs has flagged them
    if (threadIdx.x == 0) {
        p.first[s.batch] = int(groups);
        *p.count = int(groups);
    }
    __syncthreads();
    int64_t steps = 0;
    for (int64_t g0 = 0; g0 < groups; g0 += PLAN_CTA) {
        const int64_t g = g0 + threadIdx.x;
        int64_t n = 0, total;
        if (g < groups) {
            int lo = 0, hi = s.batch;  // the last b with first[b] <= g
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (p.first[mid] <= g) lo = mid;
                else hi = mid;
            }
            const Group x = group_of(seq_at(s, c, lo), a, lo, int(g - p.first[lo]));
            p.group[g] = x;
            n = (int64_t(x.steps) + OVERHEAD) * c.heads;
        }
        const int64_t at = steps + block_scan(n, warp_sum, total);
        if (g < groups) p.before[g] = at;
        steps += total;
    }
    if (threadIdx.x == 0) p.before[groups] = steps;
}

// ---- PTX ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded: false when the clock limit has passed or another role has given up; the first to give up says where.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int where) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
            *abort_flag = 1;
            atomicCAS(&g_status, 0, where);
            return false;
        }
    }
}
// The same for a whole warp, with one answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int where) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, where));
}
// One thread of the warp, known to be one.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(at)
                 : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
// Two floats at a time.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Shared-memory matrix descriptor: 128-byte swizzle, 8-row groups of 1024 bytes (stride), panels of 64 elements `leading` bytes apart.
__device__ __forceinline__ uint64_t descriptor(uint32_t at, uint32_t leading) {
    return uint64_t((at >> 4) & 0x3FFF) | uint64_t((leading >> 4) & 0x3FFF) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// Instruction descriptor, halfs with float32 accumulators, M 128: N, and whether the second operand's rows are its K index.
__host__ __device__ constexpr uint32_t instruction(int n, bool b_by_k) {
    return (1u << 4) | (b_by_k ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(TILE_ROWS >> 4) << 24);
}

template <int DP> struct Cfg {
    static constexpr int PANELS = DP / 64;  // of 64 halfs a row: 128 bytes
    static constexpr int Q_PANEL = TILE_ROWS * 128, Q_TILE = PANELS * Q_PANEL;
    static constexpr int PANEL = KEYS * 128, OPERAND = PANELS * PANEL;  // K or V of a step
    static constexpr int SMEM = 2 * Q_TILE + 2 * STAGES * OPERAND + 1024;
    static constexpr int PART = ITEM_ROWS * DP + 2 * ITEM_ROWS;
    // TMEM columns of tile t: scores of step n at 128 t + 64 (n % 2), O at O_COL + DP t
    static constexpr int O_COL = 256;
};

// What the softmax needs of a step: for each group of sixteen tokens K's scale, V's, V's power of two (minus infinity for zero) and that one's
// inverse; which groups are there, and ODD where a scale of V is no power of two (or none whose inverse is a normal number).
struct Info {
    float k[GROUPS], v_log[GROUPS], v_inv[GROUPS], v[GROUPS];
    int there;
};
constexpr int ODD = 1 << GROUPS;
__device__ __forceinline__ float power_of_two(float whole) { return __int_as_float((int(whole) + 127) << 23); }
__device__ __forceinline__ float power_in(float unit) { return float((__float_as_int(unit) >> 23) - 127); }

// The products of a step, by one thread.  `base`: the block's operands, Q of both tiles, then the stages of K, then those of V.
template <int DP> __device__ __forceinline__ void scores_of(uint32_t base, int tile, int place, int stage) {
    using C = Cfg<DP>;
    const uint64_t q = descriptor(base + tile * C::Q_TILE, 16), k = descriptor(base + 2 * C::Q_TILE + stage * C::OPERAND, 16);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
        mma_ss(128 * tile + 64 * place, q + (((i >> 2) * C::Q_PANEL + (i & 3) * 32) >> 4), k + (((i >> 2) * C::PANEL + (i & 3) * 32) >> 4), instruction(KEYS, false), i != 0);
}
template <int DP> __device__ __forceinline__ void output_of(uint32_t base, int tile, int place, int stage, bool accumulate) {
    using C = Cfg<DP>;
    const uint64_t v = descriptor(base + 2 * C::Q_TILE + (STAGES + stage) * C::OPERAND, C::PANEL);
#pragma unroll
    for (int i = 0; i < KEYS / 16; ++i)
        mma_ts(C::O_COL + DP * tile, 128 * tile + 64 * place + 8 * i, v + i * (2048 >> 4), instruction(DP, true), i != 0 || accumulate);
}

template <typename T, int FMT, int DP> __global__ void __launch_bounds__(THREADS, 1) tiles_kernel(Attn a, Cache c, Seqs s, Plan plan) {
    using C = Cfg<DP>;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[4 * STAGES + 12];
    __shared__ Info info[INFO];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_shared;
    __shared__ int found_group;
    volatile int *abort_flag = &abort_shared;
    const uint32_t base = __shfl_sync(0xffffffffu, (smem_u32(raw) + 1023u) & ~1023u, 0);
    const uint32_t q_smem = base, k_smem = base + 2 * C::Q_TILE, v_smem = k_smem + STAGES * C::OPERAND;
    const uint32_t bar0 = smem_u32(bars);
    auto k_full = [&](int i) { return bar0 + 8u * i; };
    auto k_empty = [&](int i) { return bar0 + 8u * (STAGES + i); };
    auto v_full = [&](int i) { return bar0 + 8u * (2 * STAGES + i); };
    auto v_empty = [&](int i) { return bar0 + 8u * (3 * STAGES + i); };
    auto s_full = [&](int t, int place) { return bar0 + 8u * (4 * STAGES + 2 * t + place); };
    auto p_ready = [&](int t) { return bar0 + 8u * (4 * STAGES + 4 + t); };
    auto q_ready = [&](int t) { return bar0 + 8u * (4 * STAGES + 6 + t); };
    auto o_full = [&](int t) { return bar0 + 8u * (4 * STAGES + 8 + t); };
    // the same in all threads of a warp, and known to be: what the tensor cores are told is worked out in uniform registers
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(k_full(i), 32 * CONVERTERS);
            mbar_init(k_empty(i), 2);  // one arrival for each tile
            mbar_init(v_full(i), 32 * CONVERTERS);
            mbar_init(v_empty(i), 2);
        }
        for (int t = 0; t < 2; ++t) {
            for (int i = 0; i < 2; ++i) mbar_init(s_full(t, i), 2);  // the products' completion, and the issuing thread's own arrival, behind which info is visible
            mbar_init(p_ready(t), 128);
            mbar_init(q_ready(t), 128);
            mbar_init(o_full(t), 1);
        }
        abort_shared = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    griddep_wait_cta();
    fence_before();
    __syncthreads();
    fence_after();
    // The block has all 512 columns, so they begin at 0: written so, the products' addresses are constants of the code.
    constexpr uint32_t tmem = 0;
    if (tmem_slot != 0 && threadIdx.x == 0) {
        abort_shared = 1;
        atomicCAS(&g_status, 0, S_ROOM);
    }

    // ---- this block's piece of the line ----
    Join *join = reinterpret_cast<Join *>(a.ws) + blockIdx.x;
    float *parts = reinterpret_cast<float *>(a.ws + gridDim.x * sizeof(Join));
    const int groups = *plan.count;
    const int64_t total = plan.before[groups];
    const int64_t blocks = max(int64_t(1), min(int64_t(gridDim.x), total / (OVERHEAD + 4)));
    const bool work = total > 0 && int64_t(blockIdx.x) < blocks;
    const int64_t begin = work ? total * blockIdx.x / blocks : 0, end = work ? total * (blockIdx.x + 1) / blocks : 0;
    if (threadIdx.x == 0) join->parts = 0;
    for (int g = threadIdx.x; g < groups; g += THREADS)
        if (plan.before[g] <= begin && plan.before[g + 1] > begin) found_group = g;
    __syncthreads();

    // Every role walks the same pieces: for each, its group, head and steps (none where the piece holds only units of OVERHEAD).
    struct Piece {
        Group it;
        int head, step0, steps, tiles;
        int64_t item_begin, next;  // units of the line: where the item begins, where the next piece does
    };
    int group = found_group;
    auto piece_at = [&](int64_t at) {
        Piece p;
        while (at >= plan.before[group + 1]) ++group;
        const int64_t g0 = plan.before[group];
        p.it = plan.group[group];
        const int units = p.it.steps + OVERHEAD;
        p.head = int((at - g0) / units);
        p.item_begin = g0 + int64_t(p.head) * units;
        p.next = min(end, p.item_begin + units);
        p.step0 = max(int(at - p.item_begin) - OVERHEAD, 0);
        p.steps = max(int(p.next - p.item_begin) - OVERHEAD, 0) - p.step0;
        p.tiles = p.it.rows > TILE_ROWS ? 2 : 1;
        return p;
    };

    if (warp < 8) {
        // ===== softmax of tile t: this thread has one row =====
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = uint32_t(warp & 3) * 32u << 16;
        const uint32_t s_tmem = tmem + lanes + 128 * t, o_tmem = tmem + lanes + C::O_COL + DP * t;
        uint32_t n = 0, n_s = 0;  // steps of the block; those of this tile, whose barriers' phases they count
        bool ok = true;
        for (int64_t at = begin; at < end && ok;) {
            const Piece p = piece_at(at);
            const bool starts_here = at == begin;
            at = p.next;
            if (p.steps == 0) continue;
            if (t >= p.tiles) {
                n += p.steps;
                continue;
            }
            const int row = t * TILE_ROWS + r;
            const bool live = row < p.it.rows;
            const int fr = p.it.first_row + row, i = live ? fr / a.group : 0;
            const int last = live ? int(max(min(int64_t(p.it.first) + i, int64_t(p.it.end) - 1), int64_t(-1))) : -1;  // sees keys up to here
            const int64_t after = live && a.window > 0 ? int64_t(p.it.first) + i - a.window : -(int64_t(1) << 40);   // and behind this one
            // ---- the row of Q as halfs into shared memory, a bfloat16 row divided by a power of two first ----
            float c_row = a.scale_log2;
            {
                // a warp's 32 rows come as whole lines, lanes side by side along a row, and pass through the rows' place in shared memory
                constexpr int CHUNKS = DP / 8, AT_ONCE = 32 / CHUNKS;
                const int64_t mine = (p.it.row0 + i) * a.q_stride + int64_t(p.head * a.group + (live ? fr - i * a.group : 0)) * c.dim;
                const uint32_t rows_at = q_smem + t * C::Q_TILE + (warp & 3) * (32 * 128);
                const uint16_t *q = static_cast<const uint16_t *>(a.q);
                const int ch = lane % CHUNKS;
                auto place = [&](int row, int chunk) { return rows_at + (chunk >> 3) * C::Q_PANEL + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); };
                const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
                uint4 x[CHUNKS];
#pragma unroll
                for (int k = 0; k < CHUNKS; ++k) {
                    const int row_k = k * AT_ONCE + lane / CHUNKS;
                    const int64_t at_k = __shfl_sync(0xffffffffu, mine, row_k) + ch * 8;
                    const bool in = (live_rows >> row_k & 1) && ch * 8 < c.dim;
                    x[k] = make_uint4(0, 0, 0, 0);
                    if (in && a.q_vec) x[k] = *reinterpret_cast<const uint4 *>(q + at_k);
                    else if (in) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = q[at_k + 2 * e] | uint32_t(q[at_k + 2 * e + 1]) << 16;
                        x[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
#pragma unroll
                for (int k = 0; k < CHUNKS; ++k) sts128(place(k * AT_ONCE + lane / CHUNKS, ch), x[k].x, x[k].y, x[k].z, x[k].w);
                __syncwarp();
                if constexpr (std::is_same<T, bf16>::value) {
                    __nv_bfloat162 top2 = __float2bfloat162_rn(0.f);
#pragma unroll
                    for (int k = 0; k < CHUNKS; ++k) {
                        x[k] = lds128(place(lane, k));
                        for (uint32_t w : {x[k].x, x[k].y, x[k].z, x[k].w}) top2 = __hmax2(top2, __habs2(*reinterpret_cast<__nv_bfloat162 *>(&w)));
                    }
                    const float amax = fmaxf(to_compute(top2.x), to_compute(top2.y));
                    const uint32_t e = min(max(__float_as_uint(amax) >> 23, 1u), 253u);
                    float down = 1.f;
                    if (amax > 0.f && amax < __int_as_float(0x7f800000)) {
                        down = __uint_as_float((254u - e) << 23);
                        c_row *= __uint_as_float(e << 23);
                    }
#pragma unroll
                    for (int k = 0; k < CHUNKS; ++k) {
                        uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
                        for (int d = 0; d < 4; ++d) w[d] = half2_bits(__uint_as_float(w[d] << 16) * down, __uint_as_float(w[d] & 0xFFFF0000u) * down);
                        sts128(place(lane, k), w[0], w[1], w[2], w[3]);
                    }
                }
            }
            fence_async_smem();
            fence_before();  // the reads of O of the item before
            mbar_arrive(q_ready(t));
            const int tile_first = int(min(int64_t(p.it.first) + (p.it.first_row + t * TILE_ROWS) / a.group, int64_t(p.it.end) - 1));  // least `last` of the tile
            const int64_t tile_after = a.window > 0 ? int64_t(p.it.first) + (p.it.first_row + min(p.it.rows, (t + 1) * TILE_ROWS) - 1) / a.group - a.window : -1;

            // The row's maxima: m, and d as 2^(d - 7) and m + d.  Where m is so large that a scale's power is not exact beside it, m + d is minus
            // infinity: each step then goes the long way.
            float m = LOWEST, unit = power_of_two(D_LEAST - UP), big = LOWEST + D_LEAST;
            uint64_t l2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
            for (int step = 0; step < p.steps; ++step, ++n, ++n_s) {
                const int j0 = p.it.lo + (p.step0 + step) * KEYS, place = n_s & 1;
                const uint32_t here = s_tmem + 64 * place;
                if (!warp_wait(s_full(t, place), (n_s >> 1) & 1, abort_flag, S_SCORES)) { ok = false; break; }
                fence_after();
                const Info &f = info[n % INFO];
                const int there = f.there;
                const bool masked = j0 + KEYS - 1 > tile_first || j0 <= tile_after || (there & (ODD - 1)) != ODD - 1;  // the same in all threads
                // the columns of a run of 32 that this row sees, a bit each
                auto seen = [&](int col) {
                    const int hi = min(max(last - j0 - col + 1, 0), 32), lo = int(min(max(after - j0 - col + 1, int64_t(0)), int64_t(32)));
                    const uint32_t up_to = hi == 32 ? ~0u : (1u << hi) - 1, before = lo == 32 ? ~0u : (1u << lo) - 1;
                    const uint32_t have = ((there >> (col >> 4)) & 1 ? 0xFFFFu : 0u) | ((there >> ((col >> 4) + 1)) & 1 ? 0xFFFF0000u : 0u);
                    return up_to & ~before & have;
                };
                auto hide = [&](uint32_t (&x)[32], int col) {
                    const uint32_t bits = seen(col);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(bits >> e & 1)) x[e] = __float_as_uint(NEG_INF);
                };
                // From a score of group g to its exponent.  Hidden scores are infinite before they are multiplied: the factor is never zero, however
                // small the row and the keys' scale are (a score that the least normal number stands for is zero beside any other).
                auto factor = [&](int g) { return fmaxf(c_row * f.k[g], 1.17549435e-38f); };
                float top_of[GROUPS], top = NEG_INF, top_v = NEG_INF;  // of a group's scores, the row's, and the row's with the values' scales
                auto largest = [&](const uint32_t (&x)[32], int col) {
                    float v[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        v[g] = fmaxf(__uint_as_float(x[8 * g]), __uint_as_float(x[8 * g + 1]));
#pragma unroll
                        for (int e = 2; e < 8; ++e) v[g] = fmaxf(v[g], __uint_as_float(x[8 * g + e]));
                    }
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float s = __fmul_rn(fmaxf(v[2 * g], v[2 * g + 1]), factor((col >> 4) + g));
                        top_of[(col >> 4) + g] = s;
                        top = fmaxf(top, s);
                        top_v = fmaxf(top_v, s + f.v_log[(col >> 4) + g]);
                    }
                };
                // ---- the row's largest score ----
                uint32_t x[2][32];
                tmem_ld32(here, x[0]);
                tmem_ld32(here + 32, x[1]);
                wait_ld();
                if (masked) {
                    hide(x[0], 0);
                    hide(x[1], 32);
                }
                largest(x[0], 0);
                largest(x[1], 32);
                bool o_known = step == 0, stored = false;
                // ---- weights, over the scores that have been read ----
                // One exponential y = 2^(x - m + a), a = log2(s) - d + 7, is what multiplies the codes; the sum gets y * 2^-a.  So that y is not lost where
                // the sum needs it, a is -CAP at least: below that, what multiplies the codes is zero as a half either way.
                auto lower = [&](int g) { return fminf(unit * f.v_inv[g], CAP_INVERSE); };
                const bool rise = top > m + LAG || !(top_v < big + LAG);
                if (__any_sync(0xffffffffu, rise) || there >= ODD) {
                    Maxima most{m, power_in(unit) + UP};
                    float by_l, by;
                    most.rise(top, [&](float m) {
                        float v = NEG_INF;
#pragma unroll
                        for (int g = 0; g < GROUPS; ++g) v = fmaxf(v, top_of[g] - m + f.v_log[g]);
                        return v;
                    }, by_l, by);
                    m = most.m;
                    unit = power_of_two(most.d - UP);
                    const bool huge = fabsf(m) > 4194304.f && m != LOWEST;
                    big = huge ? NEG_INF : m + most.d;
#pragma unroll
                    for (int e = 0; e < 2; ++e) l2[e] = fma2(l2[e], pair(by_l, by_l), pair(0.f, 0.f));
                    if (step > 0 && __any_sync(0xffffffffu, by != 1.f)) {
                        if (!warp_wait(o_full(t), (n_s - 1) & 1, abort_flag, S_OUTPUT)) { ok = false; break; }  // the product of the step before
                        fence_after();
                        o_known = true;
#pragma unroll 1
                        for (int d = 0; d < DP; d += 16) {
                            uint32_t y[16];
                            tmem_ld16(o_tmem + d, y);
                            wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * by);
                            tmem_st16(o_tmem + d, y);
                        }
                    }
                    if (__any_sync(0xffffffffu, huge) || there >= ODD) {  // the long way: m is subtracted from the rounded score, then a joins them
#pragma unroll 1
                        for (int g = 0; g < GROUPS; ++g) {  // a group's weights lie where its own scores and those of the groups in front of it were
                            uint32_t z[16], w[8];
                            tmem_ld16(here + 16 * g, z);
                            wait_ld();
                            const uint32_t bits = masked ? seen(16 * g) : ~0u;
                            const float s = f.v_log[g] == NEG_INF ? NEG_INF : log2f(f.v[g]);
                            const float cg = factor(g), a = fmaxf(s + (UP - most.d), -CAP), ig = fminf(unit * exp2f(-s), CAP_INVERSE);
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                float y[2];
#pragma unroll
                                for (int k = 0; k < 2; ++k)
                                    y[k] = bits >> (e + k) & 1 ? exp2_approx(__fmul_rn(__uint_as_float(z[e + k]), cg) - m + a) : 0.f;
                                l2[(e >> 1) & 1] = fma2(pair(y[0], y[1]), pair(ig, ig), l2[(e >> 1) & 1]);
                                w[e / 2] = half2_bits(y[0], y[1]);
                            }
                            tmem_st8(here + 8 * g, w);
                        }
                        stored = true;
                    }
                }
                if (!stored) {
                    const float base = UP - big, least = -CAP - m;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t w[16];
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float cg = factor(2 * q + g), mg = fmaxf(f.v_log[2 * q + g] + base, least), ig = lower(2 * q + g);
                            const uint64_t c2 = pair(cg, cg), m2 = pair(mg, mg), i2 = pair(ig, ig);
#pragma unroll
                            for (int e = 16 * g; e < 16 * g + 16; e += 2) {
                                float y0, y1;
                                unpair(fma2(pair(__uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1])), c2, m2), y0, y1);
                                y0 = exp2_approx(y0);
                                y1 = exp2_approx(y1);
                                l2[(e >> 1) & 1] = fma2(pair(y0, y1), i2, l2[(e >> 1) & 1]);
                                w[e / 2] = half2_bits(y0, y1);
                            }
                        }
                        tmem_st16(here + 16 * q, w);
                    }
                }
                wait_st();
                // Each step sees the product of the step before complete, before it lets its own begin: so no wait on this barrier is two of
                // its phases away.
                if (!o_known && !warp_wait(o_full(t), (n_s - 1) & 1, abort_flag, S_OUTPUT)) { ok = false; break; }
                fence_before();
                mbar_arrive(p_ready(t));
            }
            if (!ok) break;
            // ---- the way out ----
            if (!warp_wait(o_full(t), (n_s - 1) & 1, abort_flag, S_OUTPUT)) { ok = false; break; }  // the product of the last step
            fence_after();
            float l0, l1, l3, l4;
            unpair(l2[0], l0, l1);
            unpair(l2[1], l3, l4);
            const float sum = (l0 + l1) + (l3 + l4);
            const Out by = way_out(power_in(unit) + UP, sum);
            auto result = [&](uint32_t x) { return __uint_as_float(x) * by.first * by.second; };
            const bool whole = p.step0 == 0 && p.steps == p.it.steps;
            float *part = parts + (int64_t(blockIdx.x) * 2 + (p.step0 == 0 ? 1 : 0)) * C::PART;
            if (!whole) {
                if (live) {
                    part[ITEM_ROWS * DP + row] = m;
                    part[ITEM_ROWS * DP + ITEM_ROWS + row] = sum;
                }
#pragma unroll 1
                for (int d = 0; d < DP; d += 32) {
                    uint32_t x[32];
                    tmem_ld32(o_tmem + d, x);
                    wait_ld();
                    if (!live) continue;
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4 *>(part + row * DP + d + e) = make_float4(result(x[e]), result(x[e + 1]), result(x[e + 2]), result(x[e + 3]));
                }
            } else {
                // through the place of the warp's rows of Q, which all products have read, and out as whole lines
                constexpr int CHUNKS = DP / 8, AT_ONCE = 32 / CHUNKS;
                const uint32_t rows_at = q_smem + t * C::Q_TILE + (warp & 3) * (32 * 128);
                auto place = [&](int row, int chunk) { return rows_at + (chunk >> 3) * C::Q_PANEL + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); };
#pragma unroll 1
                for (int d = 0; d < DP; d += 32) {
                    uint32_t x[32];
                    tmem_ld32(o_tmem + d, x);
                    wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float lo = result(x[e + 2 * k]), hi = result(x[e + 2 * k + 1]);
                            if constexpr (std::is_same<T, f16>::value) w[k] = half2_bits(lo, hi);
                            else {
                                const __nv_bfloat162 b2 = __floats2bfloat162_rn(lo, hi);
                                w[k] = *reinterpret_cast<const uint32_t *>(&b2);
                            }
                        }
                        sts128(place(lane, (d + e) >> 3), w[0], w[1], w[2], w[3]);
                    }
                }
                __syncwarp();
                const int64_t mine = (p.it.row0 + i) * a.out_stride + int64_t(p.head * a.group + (live ? fr - i * a.group : 0)) * c.dim;
                uint16_t *out = static_cast<uint16_t *>(a.out);
                const int ch = lane % CHUNKS;
                const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
#pragma unroll 4
                for (int k = 0; k < CHUNKS; ++k) {
                    const int row_k = k * AT_ONCE + lane / CHUNKS;
                    const int64_t at_k = __shfl_sync(0xffffffffu, mine, row_k) + ch * 8;
                    const uint4 v = lds128(place(row_k, ch));
                    if (!(live_rows >> row_k & 1) || ch * 8 >= c.dim) continue;
                    if (a.out_vec) __stcs(reinterpret_cast<uint4 *>(out + at_k), v);
                    else {
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < 8; ++e) out[at_k + e] = uint16_t(w[e >> 1] >> (16 * (e & 1)));
                    }
                }
                __syncwarp();  // the rows are the next item's
            }
            // the item's first steps are the block before's: here is where it is joined
            if (threadIdx.x == 0 && starts_here && p.step0 > 0 && total * (int64_t(blockIdx.x) - 1) / blocks - p.item_begin <= OVERHEAD) {
                join->row0 = p.it.row0;
                join->first_row = p.it.first_row;
                join->rows = p.it.rows;
                join->head = p.head;
                join->parts = int(((p.item_begin + p.it.steps + OVERHEAD) * blocks - 1) / total) - int(blockIdx.x) + 2;
            }
        }
    } else if (warp < 8 + 2 * CONVERTERS) {
        // ===== codes into halfs: keys or values =====
        const bool is_v = warp >= 8 + CONVERTERS;
        const int sub = (warp - 6) % CONVERTERS;  // the first warp, which has the steps' info to see to as well, has no turn more than the others
        constexpr int PER_ROW = DP / 16, WARP_ROWS = 32 / PER_ROW, UNITS = KEYS / WARP_ROWS, TURNS = (UNITS + CONVERTERS - 1) / CONVERTERS;
        auto has = [&](int turn) { return turn + 1 < TURNS || sub < UNITS - CONVERTERS * (TURNS - 1); };  // the same in all threads of the warp
        // In turn i the warp takes rows WARP_ROWS * (sub + CONVERTERS * i)..., a thread sixteen codes, chunk ch of one row: eight lanes in a row are
        // four chunks of an even and an odd row, whose halfs go to different banks.
        const int ch = DP == 64 ? lane & 3 : (lane & 3) | (lane >> 3 & 1) << 2;
        const int r0 = DP == 64 ? lane >> 2 : (lane >> 2 & 1) | lane >> 4 << 1;
        const bool in_dim = ch * 16 < c.dim;
        const uint8_t *codes = (is_v ? c.v : c.k) + ch * 16;
        const uint32_t smem = (is_v ? v_smem : k_smem) + (ch >> 2) * C::PANEL;
        uint32_t n = 0;
        bool ok = true;
        for (int64_t at = begin; at < end && ok;) {
            const Piece p = piece_at(at);
            at = p.next;
            if (p.steps == 0) continue;
            // lane g of a warp (mod GROUPS) knows group g of a step: its page, and where its codes begin (-1: nowhere)
            const int32_t *table = s.table + int64_t(p.it.b) * s.cols;
            // A page's number is asked for a step before it is looked at: nothing waits for it.
            auto token_of = [&](int step) { return p.it.lo + (p.step0 + step) * KEYS + (lane % GROUPS) * 16; };
            auto seen = [&](int step, int j) { return step < p.steps && j < p.it.hi && j + 16 > p.it.first_seen; };
            auto entry_of = [&](int step) {
                const int j = token_of(step);
                return seen(step, j) ? table[j >> c.page_shift] : -1;
            };
            auto page_of = [&](int step, int32_t entry) {
                if (uint32_t(entry) < uint64_t(c.pages)) return entry;
                if (warp == 8 && lane < GROUPS && seen(step, token_of(step))) raise(a.flag, FLAG_PAGE);
                return -1;
            };
            auto begin_of = [&](int step, int32_t number) {
                const int j = token_of(step);
                return number < 0 ? int64_t(-1) : ((int64_t(number) * c.heads + p.head) * c.page + (j & (c.page - 1))) * c.dim;
            };
            uint4 x[TURNS];
            // Rows from p.it.hi on in a group that is there are read like the others: no row sees them.
            auto load = [&](int64_t offsets, int turn) {
                const int row = WARP_ROWS * (sub + CONVERTERS * turn) + r0;
                const int64_t off = __shfl_sync(0xffffffffu, offsets, (row >> 4) % GROUPS);  // a warp's rows of a turn are of one group
                if (off < 0 || !in_dim) return make_uint4(0, 0, 0, 0);
                return *reinterpret_cast<const uint4 *>(codes + off + (row & 15) * c.dim);
            };
            int32_t entry = entry_of(2), number = page_of(0, entry_of(0)), next = page_of(1, entry_of(1));
            {
                const int64_t offsets = begin_of(0, number);
#pragma unroll
                for (int turn = 0; turn < TURNS; ++turn)
                    if (has(turn)) x[turn] = load(offsets, turn);
            }
            // The scales of a step's groups, like its codes, a step ahead.
            float ks_next = 1.f, vs_next = 0.f;
            auto scales_of = [&](int32_t of) {
                ks_next = 1.f, vs_next = 0.f;
                if (warp == 8 && of >= 0) {
                    ks_next = c.k_scale[int64_t(of) * c.heads + p.head];
                    vs_next = c.v_scale[int64_t(of) * c.heads + p.head];
                }
            };
            scales_of(number);
            for (int step = 0; step < p.steps; ++step, ++n) {
                const int stage = n % STAGES;
                const bool there = number >= 0;
                const float ks = ks_next, vs = vs_next;
                scales_of(next);
                const int64_t offsets = begin_of(step + 1, next);
                if (!warp_wait(is_v ? v_empty(stage) : k_empty(stage), ((n / STAGES) & 1) ^ 1, abort_flag, S_ROOM)) { ok = false; break; }
                const uint32_t dst = smem + stage * C::OPERAND;
#pragma unroll
                for (int turn = 0; turn < TURNS; ++turn) {
                    if (!has(turn)) continue;
                    const uint32_t w[4] = {x[turn].x, x[turn].y, x[turn].z, x[turn].w};
                    x[turn] = load(offsets, turn);
                    uint32_t h[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) decode4<FMT, true>(w[e], h[2 * e], h[2 * e + 1]);
                    const int row = WARP_ROWS * (sub + CONVERTERS * turn) + r0;
                    const uint32_t at0 = dst + row * 128 + (((ch & 3) * 2 ^ (row & 7)) << 4);
                    sts128(at0, h[0], h[1], h[2], h[3]);
                    sts128(at0 ^ 16, h[4], h[5], h[6], h[7]);
                }
                if (warp == 8) {
                    const uint32_t mask = __ballot_sync(0xffffffffu, there) & ((1u << GROUPS) - 1);
                    Info &f = info[n % INFO];
                    if (lane < GROUPS) {
                        f.k[lane] = ks;
                        const bool none = vs < 1.17549435e-38f;  // a page never written
                        f.v_log[lane] = none ? NEG_INF : scale_power(vs);
                        f.v_inv[lane] = __uint_as_float(none ? 0x7F800000u : 0x7F000000u - (__float_as_uint(vs) & 0x7F800000u));
                        f.v[lane] = vs;
                    }
                    const bool odd = __any_sync(0xffffffffu, (__float_as_uint(vs) & 0x7FFFFFu) || vs > 0x1p125f);
                    if (lane == 0) f.there = int(mask) | (odd ? ODD : 0);
                }
                fence_async_smem();
                mbar_arrive(is_v ? v_full(stage) : k_full(stage));
                number = next;
                next = page_of(step + 2, entry);
                entry = entry_of(step + 3);
            }
        }
    } else if (elect_one()) {
        // ===== the products of tile t =====
        const int t = warp - (8 + 2 * CONVERTERS);
        uint32_t n = 0, n_s = 0, n_q = 0;
        bool ok = true;
        // The scores of the block's step n, the tile's step s: the keys are awaited; what info holds of the step is visible behind this
        // thread's arrival.
        auto issue_scores = [&](uint32_t n, uint32_t n_s) {
            const int stage = n % STAGES, place = n_s & 1;
            if (!mbar_wait(k_full(stage), (n / STAGES) & 1, abort_flag, S_KEYS)) return false;
            fence_after();
            scores_of<DP>(base, t, place, stage);
            commit(s_full(t, place));
            mbar_arrive(s_full(t, place));
            commit(k_empty(stage));
            return true;
        };
        for (int64_t at = begin; at < end && ok;) {
            const Piece p = piece_at(at);
            at = p.next;
            if (p.steps == 0) continue;
            if (t >= p.tiles) {
                // No rows: the tile's arrivals all the same, step by step, so that its waits never run ahead by a phase.
                for (int step = 0; step < p.steps && ok; ++step, ++n) {
                    ok = mbar_wait(k_full(n % STAGES), (n / STAGES) & 1, abort_flag, S_KEYS);
                    mbar_arrive(k_empty(n % STAGES));
                    ok = ok && mbar_wait(v_full(n % STAGES), (n / STAGES) & 1, abort_flag, S_VALUES);
                    mbar_arrive(v_empty(n % STAGES));
                }
                continue;
            }
            ok = mbar_wait(q_ready(t), n_q++ & 1, abort_flag, S_QUERIES) && issue_scores(n, n_s);
            if (p.steps > 1) ok = ok && issue_scores(n + 1, n_s + 1);
            for (int step = 0; step < p.steps && ok; ++step, ++n, ++n_s) {
                const int stage = n % STAGES;
                ok = mbar_wait(p_ready(t), n_s & 1, abort_flag, S_WEIGHTS) && mbar_wait(v_full(stage), (n / STAGES) & 1, abort_flag, S_VALUES);
                if (!ok) break;
                fence_after();
                output_of<DP>(base, t, n_s & 1, stage, step != 0);
                commit(v_empty(stage));
                commit(o_full(t));
                if (step + 2 < p.steps) ok = issue_scores(n + 2, n_s + 2);
            }
        }
        if (*abort_flag) {  // products in flight: time to end before their memory is given back
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000ll) {}
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <typename T, int FMT, int DP> int launch(const Attn &a, const Cache &c, const Seqs &s, cudaStream_t st) {
    using C = Cfg<DP>;
    static std::atomic<uint64_t> prepared{0};
    if (int e = allow_shared(tiles_kernel<T, FMT, DP>, C::SMEM, &prepared)) return e;
    const unsigned grid = unsigned(sm_count());
    const Plan plan = plan_at(a.ws + align256(grid * (sizeof(Join) + 2 * C::PART * sizeof(float))), s, a.group);
    launch_pdl(plan_kernel, dim3(1), dim3(PLAN_CTA), 0, st, a, c, s, plan);
    if (int e = check_launch("kvcache_attention (plan)")) return e;
    launch_pdl(tiles_kernel<T, FMT, DP>, dim3(grid), dim3(THREADS), C::SMEM, st, a, c, s, plan);
    if (int e = check_launch("kvcache_attention (tiles)")) return e;
    launch_pdl(join_kernel<T, DP, ITEM_ROWS>, dim3(grid, ITEM_ROWS / join_rows(ITEM_ROWS)), dim3(JOIN_CTA), 0, st, a, c);
    return check_launch("kvcache_attention (join)");
}

}  // namespace

size_t tiles_workspace(const Cache &c, const Seqs &s, int group) {
    const size_t part = c.dim <= 64 ? Cfg<64>::PART : Cfg<128>::PART;
    return align256(size_t(sm_count()) * (sizeof(Join) + 2 * part * sizeof(float))) + plan_bytes(s, group);
}

int launch_tiles(int dtype, int format, const Attn &a, const Cache &c, const Seqs &s, cudaStream_t st) {
#define DX_CALL(T, FMT) return c.dim <= 64 ? launch<T, FMT, 64>(a, c, s, st) : launch<T, FMT, 128>(a, c, s, st)
    if (dtype == DX_F16) {
        if (format == DX_CACHE_I8) DX_CALL(f16, DX_CACHE_I8);
        DX_CALL(f16, DX_CACHE_E4M3);
    }
    if (format == DX_CACHE_I8) DX_CALL(bf16, DX_CACHE_I8);
    DX_CALL(bf16, DX_CACHE_E4M3);
#undef DX_CALL
}

}  // namespace kv
}  // namespace dx

extern "C" int dx_kvcache_status(void *stream) {
    using namespace dx;
    cudaStream_t st = as_stream(stream);
    cudaError_t e = cudaStreamSynchronize(st);
    int status = 0;
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&status, kv::g_status, sizeof(int));
    if (e != cudaSuccess) return fail(DX_E_CUDA, "kvcache_status: %s", cudaGetErrorString(e));
    if (status == 0) return DX_OK;
    const int zero = 0;
    cudaMemcpyToSymbol(kv::g_status, &zero, sizeof(int));
    static const char *const where[] = {"", "keys", "values", "scores", "weights", "queries", "the output", "room for a step"};
    return fail(DX_E_CUDA, "kvcache_attention: a bounded wait for %s ran out", status < 8 ? where[status] : "?");
}
