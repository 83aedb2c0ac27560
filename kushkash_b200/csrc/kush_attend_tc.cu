// Chunk attention on the 5th-generation tensor cores (fp16 / bf16 rows, head_dim 64 or 128).
//
// A block holds up to 256 query rows of one (sequence, kv head) and walks the 128-token key tiles they see.  Two slots
// of 128 rows (M = 128 of tcgen05.mma) work in turn, so that one slot's products run under the other's softmax:
//   paired  more than 128 rows: slot i holds rows [128 i, 128 i + 128); both read every key tile
//   split   up to 128 rows (drafted tokens, short turns): both slots hold the same rows and take the key tiles in turn,
//           each with its own running maximum, sum and output; merged at the end
// Roles (16 warps of 128 registers, one block per SM): warps 0-3 and 4-7 the softmax of slots 0 and 1 (a thread per row),
// warps 8-13 bring keys and values into shared memory (16-token units in turn: records dequantized, tail and new rows
// converted; fp16), one thread of warps 14 and 15 issues the products of slots 0 and 1:
//   S[128 x 128] = Q K'^T   (both from shared memory, K-major, 128-byte swizzle), fp32 in TMEM
//   O[128 x D]  += P V      (P fp16 in TMEM over the first half of S's columns, V from shared memory, N-major)
// (softmax warps that have no rows bring keys and values too: 20 rows of drafted tokens leave six of them.)
// Keys of records enter as K' = c ks + (kb - ref), fp16, ref = the key bias of the first finished page the block sees: a shift
// of a row's scores by q ref, and large channel offsets are gone before the rounding to fp16.  The unfinished page's keys and
// the new rows enter as they are (exact for fp16, and for bf16 from 2^-17 to 65504; smaller ones as multiples of 2^-24), as q
// and new values do; q ref, in fp32, is taken off their scores.  (Shifted and rounded as the records' are they cost fp16 rows
// three quarters of their error: 7.6e-4 relative against 3.6e-4, windowed int8.)  Values of records are c vs + vb rounded to
// fp16: the products take one type of operand, and both factors apart would cost the softmax two operations a weight.  Scores,
// maxima, sums and outputs stay fp32.  The maximum m in use moves lazily: O is rescaled only when a score passes it by
// 2^TAU.  The weights enter the products as fp16, p = 2^(s - m + TC_UP) <= 2^(TAU + TC_UP) = 2^15: the upper end of fp16's
// range, so that a weight keeps its 11 bits down to 2^-23 of the row's largest and an absolute step of 2^-33 below.  (With the
// largest at 1, under a sink token whose value is near zero, the weights that make the output fell among fp16's subnormals;
// those e^-17.3 below the sink's were lost.)  Weights of a tile that the maximum moves past are rounded a second time.
// TAU = 4, 5, 6, 8 (steps 2^-35, 2^-34, 2^-33, 2^-31): ragged prefill 465, 462, 460, 455 us, windowed int8 338, 327, 325, 324.
//
// What bounds it.  A pair of 128-row tiles and a key tile are 32 products of 64 cycles (2048 cycles of tensor cores), 32768
// exponentials at 16 a cycle (2048 cycles) and 32768 dequantized values.  No unit is full: over 6000 tokens the counters show
// the tensor pipe 38% busy, the exponential pipe 38%, issue slots 44%, and waits for loads (long scoreboard, 3.9 per issued
// instruction) as the largest stall: the latency of the chain product -> softmax -> product and of the producers' loads.  One
// wave of blocks (1152 rows of 4 q heads on 8 kv heads over 30001 int4 tokens, bf16; 144 of 148 SMs) takes 622 us = 927
// TFLOP/s, 56% of the measured bf16 GEMM rate; 8192 new rows without history 616 us = 892.  (When it took 616: with the
// conversions left out 556, the softmax's arithmetic left out 497, both 449.)
// What the design rests on, each step measured on that wave or on a 2048-row chunk as it was built:
//   two slots                    one issuing warp per slot: with one for both, its waits and issue left the tensor cores idle
//                                (4200 cycles a tile for itself); operands in uniform registers (elect.sync, shuffled
//                                values): a product's issue fell from 80 to 20 cycles
//   turns of the two softmaxes   847 -> 927 TFLOP/s, passed on at half a softmax 936 (at the end 893)
//   units loaded a unit ahead    keys under the values' conversion and the other way round: 824 -> 894 TFLOP/s; a ring of
//   into registers               bulk copies in shared memory instead cost the producers more instructions than it saved
//   one pass over S              32 columns at a time; masked scores are rewritten in TMEM first (rolled loops: the code of
//                                all roles has to stay in the instruction caches; unrolled, 28% of the stalls were fetches)
//   q ref off the scores         in a loop of its own for the one tile that mixes both kinds of keys; in the masking loop it
//                                cost every row 20 to 30% (ragged prefill 557 us against 467)
//   exponentials on the FMA pipe  4, 8, 12, 16 of 32 by a polynomial: 906, 886, 865, 840 TFLOP/s; not kept
//   20 warps, registers moved    ten producing warps of 88 registers by setmaxnreg: spills, 892 TFLOP/s; not kept
// Short calls (20 rows a sequence) are bound by that chain: 64 sequences x 5 rows over 4000-8192 tokens 370 us.
//
// Waits are bounded (2 s): on a timeout the block raises the error flag, every warp leaves its loop, outputs that were not
// complete by then become NaN (a partial's maximum +inf and sum NaN, which no merge drops), and the block returns.
#include <atomic>

#include "kush_async.cuh"
#include "kush_attend.cuh"

namespace kush {

constexpr int TC_TM = 256, TC_TN = 128, TC_THREADS = 16 * WARP, TC_NPROD = 6;
constexpr float TC_TAU = 6.0f, TC_UP = 15.0f - TC_TAU;

__device__ int g_attend_error = 0;

template <int D>
struct TcSmem {
    static constexpr int BLK = 128 * 128;                    // 128 rows x 64 channels of fp16: one swizzled block
    static constexpr int TILE = BLK * (D / 64);
    static constexpr int Q = 0, K = Q + 2 * TILE, V = K + 2 * TILE, REF = V + 2 * TILE;               // REF: fp32 [D]
    static constexpr int BARS = REF + 4 * D, MISC = BARS + 8 * 16, BYTES = MISC + 16 + 1024;          // + alignment
    static_assert(BYTES <= 232448, "shared memory of a block");
};

// ------------------------------------------------------------------ tcgen05 / TMEM helpers
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    // start address, leading and stride byte offsets (16-byte units), descriptor version 1, 128-byte swizzle
    return uint64_t((addr & 0x3FFFF) >> 4) | uint64_t(lbo >> 4) << 16 | uint64_t(sbo >> 4) << 32 | uint64_t(1) << 46 |
           uint64_t(2) << 61;
}
// kind::f16: fp32 accumulators, fp16 operands, A K-major, B K-major or (n_major) N-major
__device__ __forceinline__ constexpr uint32_t instr_desc(int m, int n, bool n_major) {
    return 1u << 4 | (n_major ? 1u << 16 : 0u) | uint32_t(n >> 3) << 17 | uint32_t(m >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// the loads before it have arrived: `r`'s registers are defined from here on
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 32 columns of this warp's 32 lanes: thread = lane, register i = column i
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
            addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// byte offset of (row, 8-channel chunk) in a tile of swizzled blocks
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
    return uint32_t((chunk >> 3) * (128 * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ void st_chunk(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// The exact fp16 codes of 8 (int4: 16) channels.  int4: 8 bytes = channels 8 c .. + 7 in the low nibbles (lo), D/2 + 8 c ..
// in the high ones (hi); int8: 16 bytes = channels 16 c .. + 7 (lo) and + 8 .. + 15 (hi).
template <int BITS>
__device__ __forceinline__ void codes_of(const uint32_t (&w)[BITS / 2], uint32_t (&lo)[4], uint32_t (&hi)[4]) {
    if constexpr (BITS == 4) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t x = prmt(w[i], 0, 0x3120);             // bytes b0 b2 b1 b3
            const uint32_t y = x >> 8;                             // b2 b1 b3
            lo[2 * i] = h2_sub(and_xor(x, 0x000F000Fu, 0x64086408u), 0x64086408u);
            lo[2 * i + 1] = h2_sub(and_xor(y, 0x000F000Fu, 0x64086408u), 0x64086408u);
            hi[2 * i] = h2_fma(and_xor(x, 0x00F000F0u, 0x64806480u), 0x2C002C00u, 0xD480D480u);
            hi[2 * i + 1] = h2_fma(and_xor(y, 0x00F000F0u, 0x64806480u), 0x2C002C00u, 0xD480D480u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t u = w[i] ^ 0x80808080u;                 // signed code -> c + 128
            uint32_t(&o)[4] = i < 2 ? lo : hi;
            o[2 * (i & 1)] = h2_sub(prmt(u, 0x64646464u, 0x5140), 0x64806480u);
            o[2 * (i & 1) + 1] = h2_sub(prmt(u, 0x64646464u, 0x7342), 0x64806480u);
        }
    }
}

template <class T>
__device__ __forceinline__ void load_words(const uint8_t* p, T* w, int n) {          // n words (2 or 4), aligned to them
    if (n == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x;
        w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    }
}

// A 16-token unit of a key tile for one warp: lane = (row group rg, column c) holds rows rg, rg + RG, ..., BPL bytes each.
template <int D, int BITS, int P>
struct Unit {
    using F = Fmt<D, BITS, P>;
    static constexpr int W = BITS / 2, BPL = 4 * W, LPR = F::DC / BPL, RG = WARP / LPR, RPL = 16 / RG;
};

// a packed unit's bytes into L2, ahead of their loads (16-byte address and size)
__device__ __forceinline__ void bulk_to_l2(const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ bool mbar_done(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok;
}
// the rest of a wait: the warp sleeps in try_wait for up to 20 us at a time (polls would take issue slots from the
// softmax); `limit` ns without the phase and the block gives up
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int* gave_up, uint64_t limit) {
    uint64_t t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(ok)
            : "r"(bar), "r"(parity), "r"(20000)
            : "memory");
        if (ok) return true;
        if (*gave_up) return false;
        uint64_t now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (t0 == 0) t0 = now;
        else if (now - t0 > limit) {
            *gave_up = 1;
            atomicExch(&g_attend_error, 1);
            return false;
        }
    }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// grid (row tiles, Hkv, n_splits), block 512.  HELD: one slot keeps back one tile's weights (a.held), so that waits run out.
template <int D, int BITS, int P, class IN, bool HELD>
__global__ void __launch_bounds__(TC_THREADS, 1) attend_tc_kernel(AttendArgs a) {
    using F = Fmt<D, BITS, P>;
    using U = Unit<D, BITS, P>;
    using M = TcSmem<D>;
    constexpr int CH = D / 8;                                      // 8-channel chunks of a row
    extern __shared__ uint8_t smem_raw[];
    pdl_wait();
    const int tid = threadIdx.x, wid = tid / WARP, lane = tid % WARP;
    const int h = blockIdx.y, z = blockIdx.z;
    RowTile t;
    if (!row_tile(a, int(gridDim.x) - 1 - int(blockIdx.x), TC_TM, t)) return;      // later rows, more keys: first
    const KeyTiles kt = key_tiles(t.p0, t.p1, a.window, a.sinks, TC_TN);
    int i0, i1;
    key_split(a, z, TC_TM, TC_TN, kt.count, i0, i1);
    auto grow = [&](int r) { return t.q0 + (t.r0 + r) / a.G; };                    // global row of tile row r
    auto ghead = [&](int r) { return (t.r0 + r) % a.G; };                          // its q head in the group
    if (i0 >= i1) {                                                                // (n_splits > 1) empty partials
        for (int r = tid; r < t.nr; r += TC_THREADS) {
            float* ml = a.part_ml + 2 * part_row(a, grow(r), h, z, ghead(r));
            ml[0] = -INFINITY;
            ml[1] = 0.0f;
        }
        return;
    }
    const bool paired = t.nr > 128;
    // softmax warps with rows, of slot 0 and 1; the others join the producers
    const int rows0 = (min(t.nr, 128) + WARP - 1) / WARP, rows1 = paired ? (t.nr - 128 + WARP - 1) / WARP : rows0;
    const int n_prod = TC_NPROD + 8 - rows0 - rows1;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - smem_u32(smem_raw));
    float* ref = reinterpret_cast<float*>(sm + M::REF);
    const uint32_t bars = base + M::BARS;
    const uint32_t k_full = bars, k_empty = bars + 16, v_full = bars + 32, v_empty = bars + 48, s_full = bars + 64,
                   p_full = bars + 80, o_full = bars + 96, turn = bars + 112;      // pairs: [stage] or [slot]
    volatile int* gave_up = reinterpret_cast<volatile int*>(sm + M::MISC);
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(sm + M::MISC + 4);
    if (tid == 0) {
        uint64_t* b = reinterpret_cast<uint64_t*>(sm + M::BARS);
        const int count[8] = {8, 2, 8, 2, 1, 0, 1, 0};                             // (0: a slot's warps)
        for (int i = 0; i < 16; i++) mbar_init(b + i, count[i / 2] ? count[i / 2] : i & 1 ? rows1 : rows0);
        *gave_up = 0;
        fence_mbar_init();
    }
    if (wid == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // bounded wait for the phase of `parity` of a barrier; false if this block gave up
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        return mbar_done(bar, parity) || wait_long(bar, parity, gave_up, HELD ? a.held.limit_ms * 1000000ull : 2000000000ull);
    };
    const int32_t* bt = a.block_table + int64_t(t.s) * a.max_pages;
    const uint8_t* hcache = a.cache + int64_t(h) * a.head_stride;
    const int full = t.ctx / P * P;                                                // cached tokens in finished pages
    // the key reference: the bias of the first finished page that the row tile sees (the same for all its splits)
    const int first = kt.ns > 0 ? 0 : kt.lo / P * P;
    const bool have_ref = first < full;
    if (tid < D) {
        const uint8_t* rec = have_ref ? hcache + int64_t(bt[first / P]) * a.block_stride : nullptr;
        ref[tid] = have_ref ? h_load(rec + F::OFF_KB, tid) : 0.0f;
    }
    // query rows to fp16, negated under a negative scale (the softmax multiplies by its magnitude)
    {
        const IN* q = static_cast<const IN*>(a.q);
        const float sign = a.sm_log2 < 0.0f ? -1.0f : 1.0f;
        for (int i = tid; i < t.nr * CH; i += TC_THREADS) {
            const int r = i / CH, c = i % CH;
            const uint4 raw = *reinterpret_cast<const uint4*>(q + grow(r) * a.q_stride + int64_t(h * a.G + ghead(r)) * D + 8 * c);
            const IN* e = reinterpret_cast<const IN*>(&raw);
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = pack_h2(sign * to_f32(e[2 * j]), sign * to_f32(e[2 * j + 1]));
            st_chunk(base + M::Q + (r >> 7) * M::TILE + tile_off(r & 127, c), w[0], w[1], w[2], w[3]);
        }
    }
    fence_async();
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_at;
    // Whether a slot works on the key tile of index it.  Split: in turn.  Paired: some row of the slot sees a token of it:
    // slot 0 (whose last row is mid0) the tiles up to end0, slot 1 (whose first row is mid0 or mid0 + 1) all but the window
    // tiles [gap0, gap1) behind the sinks that only slot 0's rows reach back to.
    int end0 = i1, gap0 = 0, gap1 = 0;
    if (paired) {
        const int mid0 = t.ctx + (t.r0 + 127) / a.G, mid1 = t.ctx + (t.r0 + 128) / a.G;
        const int lo1 = a.window > 0 ? max(0, mid1 - a.window + 1) : 0;
        end0 = min(i1, kt.a + mid0 / TC_TN + 1 - kt.b);                            // (mid0 >= lo: a window tile)
        gap0 = kt.a + (a.sinks > kt.b * TC_TN ? (min(a.sinks, lo1) + TC_TN - 1) / TC_TN - kt.b : 0);
        gap1 = kt.a + lo1 / TC_TN - kt.b;                                          // (lo1 <= mid1, a tile of the list)
    }
    auto active = [&](int slot, int it) -> bool {
        if (!paired) return ((it - i0) & 1) == slot;
        return slot == 0 ? it < end0 : it < gap0 || it >= gap1;
    };
    bool ok = true;

    if (wid < 8 && (wid & 3) < (wid < 4 ? rows0 : rows1)) {
        // ---------------------------------------------------------------- softmax: thread = row of its slot
        const int slot = wid >> 2, row = (wid & 3) * WARP + lane, wrow = (wid & 3) * WARP;
        const int r = paired ? slot * 128 + row : row;                             // tile row
        const int pos = t.ctx + (t.r0 + min(r, t.nr - 1)) / a.G;
        const int wp0 = __shfl_sync(0xffffffffu, pos, 0), wp1 = __shfl_sync(0xffffffffu, pos, 31);
        const float sc = fmaxf(fabsf(a.sm_log2), 1e-30f);                          // (a masked score stays -inf under scale 0)
        const uint32_t lanes = uint32_t(wrow) << 16;
        const uint32_t s_at = tmem + lanes + 128 * slot, o_at = tmem + lanes + 256 + 128 * slot;
        float qref = 0.0f;                                                         // q ref: the shift of the records' scores
        if (have_ref) {
            const uint8_t* qr = sm + M::Q + (paired ? slot * M::TILE : 0);
#pragma unroll 1
            for (int c = 0; c < CH; c++) {
                const uint4 raw = *reinterpret_cast<const uint4*>(qr + tile_off(row, c));
                const __half2* e = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 x = __half22float2(e[i]);
                    qref = fmaf(x.x, ref[8 * c + 2 * i], qref);
                    qref = fmaf(x.y, ref[8 * c + 2 * i + 1], qref);
                }
            }
        }
        float m = -INFINITY;                                                       // the maximum in use, log2 units
        float2 la = make_float2(0.0f, 0.0f), lb = la;                              // the weights' sum, in four parts
        int n = 0;                                                                 // tiles done by this slot
        // Paired slots take turns: both softmaxes at once would leave the tensor cores idle and then wait for them together.
        // Slot 0's tile goes before slot 1's, slot 1's before slot 0's next; a tile that a slot has no part in passes on.
        auto pass_on = [&] {
            if (paired && lane == 0) bar_arrive(turn + 8 * slot);
        };
        for (int it = i0; it < i1; it++) {
            const int nt = it - i0;
            const bool work = active(slot, it);
            ok = !work || wait(s_full + 8 * slot, n & 1);
            if (paired) ok = ok && (slot == 1 ? wait(turn, nt & 1) : nt == 0 || wait(turn + 8, (nt - 1) & 1));
            ok = __all_sync(0xffffffffu, ok);                                      // (converged: tcgen05.ld is warp-aligned)
            if (!ok) break;
            if (!work) {
                pass_on();
                continue;
            }
            fence_after();
            {
                const int j0 = kt.tile(it) * TC_TN;
                // columns [0, hi] seen, and of those [lo, ...) or [0, sk)
                const int hi = pos - j0, lo = a.window > 0 ? pos - a.window + 1 - j0 : -1, sk = a.sinks - j0;
                // columns from `exact` on hold unshifted keys: q ref comes off them here, or (all columns) with the maximum
                const int exact = have_ref ? full - j0 : TC_TN;
                const float shift = exact <= 0 ? -qref * sc : 0.0f;
                const bool cut = j0 + TC_TN - 1 > wp0 || (a.window > 0 && j0 < wp1 - a.window + 1 && j0 + TC_TN > a.sinks);
                // (loops over 32-column pieces stay rolled: five roles' code shares the instruction caches)
                if (exact > 0 && exact < TC_TN) {                                  // once in a row's walk
#pragma unroll 1
                    for (int c = exact / 32; c < 4; c++) {
                        uint32_t x[32];
                        tmem_ld32(s_at + 32 * c, x);
                        wait_ld(x);
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (32 * c + i >= exact) x[i] = __float_as_uint(__uint_as_float(x[i]) - qref);
                        tmem_st32(s_at + 32 * c, x);
                    }
                    wait_st();
                }
                if (cut) {                                                         // masked scores become -inf in TMEM
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t x[32];
                        tmem_ld32(s_at + 32 * c, x);
                        wait_ld(x);
                        const int h0 = hi - 32 * c, l0 = lo - 32 * c, k0 = sk - 32 * c;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (i > h0 || (i < l0 && i >= k0)) x[i] = 0xFF800000u;
                        tmem_st32(s_at + 32 * c, x);
                    }
                    wait_st();
                }
                // One pass: 32 columns at a time, the next ones on their way from TMEM; the maximum in use moves when a piece
                // passes it by 2^TAU (seldom after a row's first tile), and then takes O, the sum and this tile's earlier
                // weights along.
                auto move_max = [&](int c, float mx) {
                    const bool up = mx > m + TC_TAU;
                    const float corr = up ? fast_exp2(m - mx) : 1.0f;                    // first scores: 2^-inf = 0
                    if (up) m = mx;
                    la = __fmul2_rn(la, make_float2(corr, corr));
                    lb = __fmul2_rn(lb, make_float2(corr, corr));
#pragma unroll 1
                    for (int e = 0; e < (n > 0 ? D / 32 : 0); e++) {               // O (the slot's last product is done)
                        uint32_t x[32];
                        tmem_ld32(o_at + 32 * e, x);
                        wait_ld(x);
#pragma unroll
                        for (int i = 0; i < 32; i++) x[i] = __float_as_uint(__uint_as_float(x[i]) * corr);
                        tmem_st32(o_at + 32 * e, x);
                    }
                    wait_st();                                                     // (read back below)
#pragma unroll 1
                    for (int e = 0; e < c; e++) {                                  // P's pieces before this one
                        uint32_t x[32], p[16];
                        tmem_ld32(s_at + 16 * e, x);
                        wait_ld(x);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
                            p[i] = pack_h2(w.x * corr, w.y * corr);            // (corr itself may be below fp16's range)
                        }
                        tmem_st16(s_at + 16 * e, p);
                        wait_st();
                    }
                };
                auto top = [&](const uint32_t (&x)[32]) -> float {                 // the piece's largest score, log2 units
                    float m4[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) m4[i] = fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 4]));
#pragma unroll
                    for (int i = 8; i < 32; i += 8)
#pragma unroll
                        for (int k = 0; k < 4; k++) m4[k] = max3(m4[k], __uint_as_float(x[i + k]), __uint_as_float(x[i + k + 4]));
                    return fmaf(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), sc, shift);
                };
                // the weights of piece c in place of its scores (first the differences, then all 32 exponentials without a
                // dependence between them, under which the next piece's maximum is taken), its sum and its P
                auto piece = [&](int c, uint32_t (&x)[32], uint32_t (&y)[32], float mx, auto last) -> float {
                    if (__any_sync(0xffffffffu, mx > m + TC_TAU)) move_max(c, mx); // (m = -inf: any score)
                    const float mm = m == -INFINITY ? 0.0f : TC_UP - m + shift;    // nothing seen yet: weights 0
                    const float2 sc2 = make_float2(sc, sc), mm2 = make_float2(mm, mm);
                    if constexpr (!decltype(last)::value) tmem_ld32(s_at + 32 * c + 32, y);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 d = __ffma2_rn(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, mm2);
                        x[i] = __float_as_uint(d.x);
                        x[i + 1] = __float_as_uint(d.y);
                    }
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = __float_as_uint(fast_exp2(__uint_as_float(x[i])));
                    float next = 0.0f;
                    if constexpr (!decltype(last)::value) {
                        wait_ld(y);
                        next = top(y);
                    }
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 e = make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
                        if (i & 1) lb = __fadd2_rn(lb, e);
                        else la = __fadd2_rn(la, e);
                        p[i] = pack_h2(e.x, e.y);
                    }
                    tmem_st16(s_at + 16 * c, p);
                    return next;
                };
                uint32_t x[32], y[32];
                tmem_ld32(s_at, x);
                wait_ld(x);
                float mx = piece(0, x, y, top(x), IC<0>{});
                mx = piece(1, y, x, mx, IC<0>{});
                pass_on();                                                         // (half of it left: the exponentials of both overlap)
                mx = piece(2, x, y, mx, IC<0>{});
                piece(3, y, x, mx, IC<1>{});
                wait_st();
            }
            fence_before();
            __syncwarp();
            if (lane == 0 && !(HELD && slot == a.held.slot && n == a.held.tile)) bar_arrive(p_full + 8 * slot);
            n++;
        }
        // ---------------------------------------------------------------- the slot's output
        float l = (la.x + la.y) + (lb.x + lb.y);
        if (ok && n > 0) {
            ok = __all_sync(0xffffffffu, wait(o_full + 8 * slot, 0));
            fence_after();
        }
        // split: slot 1 hands its maximum, sum and output over (in the key buffers and, at 128 channels, the first value buffer's
        // front; no longer read)
        float* xm = reinterpret_cast<float*>(sm + M::K);                           // [2][128] m, l
        float* xo = xm + 256;                                                      // [128][D + 4]
        if (!paired) {
            // both slots' products are done before the key buffers are reused
            if (ok && slot == 1) ok = __all_sync(0xffffffffu, wait(o_full, 0));
            if (slot == 1) {
                xm[row] = n > 0 ? m : -INFINITY;
                xm[128 + row] = l;
                if (n > 0 && ok) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t x[32];
                        tmem_ld32(o_at + 32 * c, x);
                        wait_ld(x);
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4*>(xo + row * (D + 4) + 32 * c + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                    }
                }
            }
            asm volatile("bar.sync 1, %0;" ::"r"(2 * WARP * rows0) : "memory");
        }
        // (another warp of the block gave up: o_full may have come without the last products, xo from slot 1 not at all)
        ok = __all_sync(0xffffffffu, ok && *gave_up == 0);
        if (paired || slot == 0) {
            float mo = -INFINITY, f0 = 1.0f, f1 = 0.0f;
            if (!paired) {
                mo = xm[row];
                const float mn = fmaxf(m, mo);
                f0 = m == -INFINITY ? 0.0f : fast_exp2(m - mn);
                f1 = mo == -INFINITY ? 0.0f : fast_exp2(mo - mn);
                l = l * f0 + (f1 > 0.0f ? xm[128 + row] * f1 : 0.0f);
                m = mn;
            }
            const bool real = r < t.nr;
            const int64_t pr = real ? part_row(a, grow(r), h, z, ghead(r)) : 0;
            const float inv = a.n_splits > 1 ? 1.0f : l > 0.0f ? 1.0f / l : 0.0f;
            IN* o = real ? static_cast<IN*>(a.out) + ((grow(r) * a.H + h) * a.G + ghead(r)) * D : nullptr;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t x[32];
                if (n > 0 && ok) {
                    tmem_ld32(o_at + 32 * c, x);
                    wait_ld(x);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = ok ? 0u : 0x7FC00000u;
                }
                float y[32];
#pragma unroll
                for (int i = 0; i < 32; i++) y[i] = __uint_as_float(x[i]) * f0;
                if (!paired && f1 > 0.0f) {
#pragma unroll
                    for (int i = 0; i < 32; i++) y[i] = fmaf(f1, xo[row * (D + 4) + 32 * c + i], y[i]);
                }
                if (!real) continue;
                if (a.n_splits > 1) {
                    float4* po = reinterpret_cast<float4*>(a.part_o + pr * D + 32 * c);
#pragma unroll
                    for (int i = 0; i < 8; i++) po[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        alignas(16) IN e[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) e[j] = from_f32<IN>(y[i + j] * inv);
                        *reinterpret_cast<uint4*>(o + 32 * c + i) = *reinterpret_cast<const uint4*>(e);
                    }
                }
            }
            if (real && a.n_splits > 1) {
                // sum and output are in units of 2^(m - TC_UP); log2 units -> natural, for the combine
                const bool whole = ok && l == l;                                  // (NaN scores leave m as it was)
                a.part_ml[2 * pr] = whole ? (m - TC_UP) * 0.69314718055994531f : INFINITY;
                a.part_ml[2 * pr + 1] = whole ? l : NAN;
            }
        }
        fence_before();
    } else if (wid < 8 + TC_NPROD) {                                               // (and softmax warps without rows)
        // ---------------------------------------------------------------- keys and values into shared memory
        // Work comes in units of 16 tokens, keys and values: 8 of a tile, then the next tile's; this warp's k-th unit is
        // x = w + n_prod k.  Where its units come from is worked out for 32 of them at a time, a lane each, which also asks for
        // their bytes into L2.  A unit's keys are converted, then the next unit's keys loaded into the same registers, under
        // the conversion of the values, and the other way round.
        const int w = wid >= 8 ? wid - 8 : TC_NPROD + (wid < 4 ? wid - rows0 : 4 - rows0 + (wid & 3) - rows1);
        const int units = 8 * (i1 - i0), mine = w < units ? (units - w + n_prod - 1) / n_prod : 0;
        auto batch = [&](int i, int32_t& f, int32_t& bl) {                         // token | kind, and the packed unit's block
            const int k = 32 * i + lane, x = w + n_prod * k;
            f = bl = 0;
            if (k < mine) {
                const int j0 = kt.tile(i0 + (x >> 3)) * TC_TN + 16 * (x & 7);
                // 0 no row sees a token of it, 1 packed, 2 new rows, 3 mixed
                const int kind = j0 > t.p1 || (j0 + 15 < kt.lo && j0 >= kt.ns) ? 0 : j0 + 16 <= full ? 1
                                 : j0 >= t.ctx && j0 + 15 <= t.p1 ? 2 : 3;
                f = j0 | kind;
                if (kind == 1) {
                    bl = bt[j0 / P];
                    const uint8_t* rec = hcache + int64_t(bl) * a.block_stride;
                    if constexpr (P == 16) {
                        bulk_to_l2(rec, F::RB);
                    } else {
                        bulk_to_l2(rec + j0 % P * F::DC, 16 * F::DC);
                        bulk_to_l2(rec + F::OFF_VQ + j0 % P * F::DC, 16 * F::DC);
                        bulk_to_l2(rec + F::OFF_KS, F::RB - F::OFF_KS);
                    }
                }
            }
        };
        int32_t from, blk, from1, blk1;                                            // of units 32 i + lane; of the next batch
        batch(0, from, blk);
        batch(1, from1, blk1);

        // packed: lane = (row group rg, column c) has rows rg, rg + RG, ... and the chunks c_a, c_b of each, in the order of
        // its stores (int8: lanes of a row's second block store their odd chunk first, so that the eight lanes of a row fall
        // in distinct banks)
        const int c = lane % U::LPR, rg = lane / U::LPR;
        const int swap = BITS == 8 && D == 128 ? c >> 2 : 0;
        const int c_a = BITS == 4 ? c : 2 * c + swap, c_b = BITS == 4 ? c + D / 16 : 2 * c + 1 - swap;
        const uint32_t at_a = tile_off(rg, c_a), at_b = tile_off(rg, c_b);         // in a unit's first rows
        const int code_a = rg * F::DC + (BITS == 4 ? 8 * c : 8 * c_a), code_b = rg * F::DC + 8 * c_b;
        uint32_t rf[8];                                                            // the reference of the lane's channels
#pragma unroll
        for (int i = 0; i < 4; i++) {
            rf[i] = pack_h2(ref[8 * c_a + 2 * i], ref[8 * c_a + 2 * i + 1]);
            rf[4 + i] = pack_h2(ref[8 * c_b + 2 * i], ref[8 * c_b + 2 * i + 1]);
        }
        // new rows: chunk cc of rows r0, r0 + RPI, ...
        constexpr int RPI = WARP / CH, NI = 16 / RPI;
        const int cc = lane % CH, r0 = lane / CH;
        const uint32_t at_r = tile_off(r0, cc);

        // registers of a unit's keys (values): packed, words [0, RPL W) codes and [16, 32) scales and biases of chunks a and
        // b (word 16: the scale of row lane or the bias of row lane - 16); new rows, the rows
        uint32_t kr[32], vr[32];
        auto load = [&](auto kvc, int32_t f, int32_t bl, uint32_t (&r)[32]) {
            constexpr bool kv = decltype(kvc)::value;
            const int j0 = f & ~15, kind = f & 15;
            if (kind == 1) {
                const uint8_t* rec = hcache + int64_t(bl) * a.block_stride;
                const uint8_t* rows = rec + (kv ? F::OFF_VQ : 0) + j0 % P * F::DC;
#pragma unroll
                for (int i = 0; i < U::RPL; i++) {
                    load_words(rows + code_a + U::RG * i * F::DC, r + U::W * i, 2);
                    if constexpr (BITS == 8) load_words(rows + code_b + U::RG * i * F::DC, r + U::W * i + 2, 2);
                }
                if constexpr (kv) {
                    r[16] = reinterpret_cast<const uint16_t*>(rec + (lane < 16 ? F::OFF_VS : F::OFF_VB))[j0 % P + (lane & 15)];
                } else {
                    load_words(rec + F::OFF_KS + 16 * c_a, r + 16, 4);
                    load_words(rec + F::OFF_KS + 16 * c_b, r + 20, 4);
                    load_words(rec + F::OFF_KB + 16 * c_a, r + 24, 4);
                    load_words(rec + F::OFF_KB + 16 * c_b, r + 28, 4);
                }
                return;
            }
            if (kind != 2) return;
            const int64_t stride = kv ? a.v_stride : a.k_stride;
            const IN* src = static_cast<const IN*>(kv ? a.v_new : a.k_new) + (t.q0 + (j0 - t.ctx + r0)) * stride + int64_t(h) * D + 8 * cc;
#pragma unroll
            for (int i = 0; i < NI; i++, src += RPI * stride) load_words(reinterpret_cast<const uint8_t*>(src), r + 4 * i, 4);
        };
        // a unit that is not of one kind (the unfinished page, its border to the new rows, tokens that no row sees, which are
        // zeros): row after row
        auto mixed = [&](auto kvc, int j0, int kind, uint32_t dst) {
            constexpr bool kv = decltype(kvc)::value;
            const int64_t stride = kv ? a.v_stride : a.k_stride;
            const IN* rows = static_cast<const IN*>(kv ? a.v_new : a.k_new) + (t.q0 + (j0 - t.ctx)) * stride + int64_t(h) * D + 8 * cc;
            const IN* tail = static_cast<const IN*>(a.tail_k) + (int64_t(a.tail_idx[t.s]) * a.H + h) * P * D + 8 * cc;
#pragma unroll 1
            for (int i = 0; i < NI; i++) {
                const int row = i * RPI + r0, j = j0 + row;
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; k++) y[k] = 0.0f;
                if (kind == 3 && kt.seen(j, t.p1)) {
                    if (j >= t.ctx || (!kv && j >= full)) {
                        const uint4 raw = *reinterpret_cast<const uint4*>(j >= t.ctx ? rows + row * stride : tail + (j % P) * D);
                        const IN* e = reinterpret_cast<const IN*>(&raw);
#pragma unroll
                        for (int k = 0; k < 8; k++) y[k] = to_f32(e[k]);
                    } else {
                        const uint8_t* rec = hcache + int64_t(bt[j / P]) * a.block_stride;
                        const int at = j % P;
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const int d = 8 * cc + k;
                            y[k] = kv ? fmaf(float(code_at<D, BITS>(rec + F::OFF_VQ + at * F::DC, d)), h_load(rec + F::OFF_VS, at),
                                             h_load(rec + F::OFF_VB, at))
                                      : fmaf(float(code_at<D, BITS>(rec + at * F::DC, d)), h_load(rec + F::OFF_KS, d),
                                             h_load(rec + F::OFF_KB, d) - ref[d]);
                        }
                    }
                }
                st_chunk(dst + tile_off(row, cc), pack_h2(y[0], y[1]), pack_h2(y[2], y[3]), pack_h2(y[4], y[5]), pack_h2(y[6], y[7]));
            }
        };
        auto convert = [&](auto kvc, int32_t f, uint32_t (&r)[32], uint32_t dst) {
            constexpr bool kv = decltype(kvc)::value;
            const int j0 = f & ~15, kind = f & 15;
            if (kind == 1) {
                if constexpr (!kv) {
#pragma unroll
                    for (int i = 0; i < 8; i++) r[24 + i] = h2_sub(r[24 + i], rf[i]);
                }
#pragma unroll
                for (int i = 0; i < U::RPL; i++) {
                    uint32_t cw[U::W], lo[4], hi[4];
#pragma unroll
                    for (int j = 0; j < U::W; j++) cw[j] = r[U::W * i + j];
                    codes_of<BITS>(cw, lo, hi);
                    if constexpr (kv) {
                        const uint32_t vs = __shfl_sync(0xffffffffu, r[16], rg + U::RG * i) * 0x10001u;
                        const uint32_t vb = __shfl_sync(0xffffffffu, r[16], 16 + rg + U::RG * i) * 0x10001u;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            lo[j] = h2_fma(lo[j], vs, vb);
                            hi[j] = h2_fma(hi[j], vs, vb);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            lo[j] = h2_fma(lo[j], r[16 + j], r[24 + j]);
                            hi[j] = h2_fma(hi[j], r[20 + j], r[28 + j]);
                        }
                    }
                    const uint32_t flip = U::RG == 4 && (i & 1) ? 64 : 0;          // rows 4 apart: the swizzle's bit 2
                    st_chunk(dst + ((at_a ^ flip) + U::RG * 128 * i), lo[0], lo[1], lo[2], lo[3]);
                    st_chunk(dst + ((at_b ^ flip) + U::RG * 128 * i), hi[0], hi[1], hi[2], hi[3]);
                }
                return;
            }
            if (kind != 2) {
                mixed(kvc, j0, kind, dst);
                return;
            }
#pragma unroll
            for (int i = 0; i < NI; i++) {
                uint32_t p[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t e = r[4 * i + k];                               // two channels
                    if constexpr (std::is_same_v<IN, __half>) p[k] = e;
                    else p[k] = pack_h2(__uint_as_float(e << 16), __uint_as_float(e & 0xFFFF0000u));
                }
                // (rows RPI apart: the swizzle's upper bits)
                const uint32_t flip = RPI == 2 ? (i & 3) << 5 : (i & 1) << 6;
                st_chunk(dst + ((at_r ^ flip) + RPI * 128 * i), p[0], p[1], p[2], p[3]);
            }
        };
        int32_t f = __shfl_sync(0xffffffffu, from, 0), bl = __shfl_sync(0xffffffffu, blk, 0);
        if (mine > 0) {
            load(IC<0>{}, f, bl, kr);
            load(IC<1>{}, f, bl, vr);
        }
#pragma unroll 1
        for (int k = 0; k < mine; k++) {
            const int x = w + n_prod * k, n = x >> 3, st = n & 1;
            const uint32_t dst = base + M::K + st * M::TILE + (x & 7) * 2048, before = ((n >> 1) - 1) & 1;
            int32_t f1 = 0, bl1 = 0;
            if (k + 1 < mine) {
                if (((k + 1) & 31) == 0) {
                    from = from1;
                    blk = blk1;
                    batch((k + 1) / 32 + 1, from1, blk1);
                }
                f1 = __shfl_sync(0xffffffffu, from, (k + 1) & 31);
                bl1 = __shfl_sync(0xffffffffu, blk, (k + 1) & 31);
            }
            // (a fresh barrier lets tiles 0 and 1 pass; a buffer that is still read is not written when a wait runs out)
            if (!__all_sync(0xffffffffu, wait(k_empty + 8 * st, before))) break;
            convert(IC<0>{}, f, kr, dst);
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(k_full + 8 * st);
            if (k + 1 < mine) load(IC<0>{}, f1, bl1, kr);
            if (!__all_sync(0xffffffffu, wait(v_empty + 8 * st, before))) break;
            convert(IC<1>{}, f, vr, dst + (M::V - M::K));
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(v_full + 8 * st);
            if (k + 1 < mine) load(IC<1>{}, f1, bl1, vr);
            f = f1;
            bl = bl1;
        }
    } else {
        // ---------------------------------------------------------------- the products: a warp for each slot
        // For each key tile S, then (P written) O: the next tile's S overwrites P, and products of one thread run in order.
        // Two warps, because one thread's waits and issue (50 cycles a product) would leave the tensor cores idle for half
        // the time; so one slot's products run under the other's.  The warp walks together on warp-uniform values (the
        // products' operands live in uniform registers), one thread issues.
        constexpr uint32_t ID_S = instr_desc(128, TC_TN, false), ID_O = instr_desc(128, D, true);
        auto uni = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
        const bool leader = elect_one();
        const int slot = uni(wid - 8 - TC_NPROD), n1 = uni(i1 - i0), pr = uni(paired);
        // tiles this slot works on: paired, all but [skip0, skip1); split, every other one
        const int skip0 = uni((slot == 0 ? end0 : gap0) - i0), skip1 = uni((slot == 0 ? i1 : gap1) - i0);
        const uint32_t s_tm = uni(tmem) + 128 * slot, o_tm = s_tm + 256;
        const uint64_t q_desc = smem_desc(base + M::Q + (pr && slot ? M::TILE : 0), 16, 1024);
        const uint64_t k_desc = smem_desc(base + M::K, 16, 1024), v_desc = smem_desc(base + M::V, M::BLK, 1024);
        auto works = [&](int n) -> bool { return pr ? n < skip0 || n >= skip1 : (n & 1) == slot; };
        auto scores = [&](int n) {                                                 // the leader: S of tile n (its keys are there)
            if (works(n)) {
                const uint64_t kd = k_desc + (n & 1) * (M::TILE >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const uint32_t off = ((k >> 2) * M::BLK + (k & 3) * 32) >> 4;
                    mma_ss(s_tm, q_desc + off, kd + off, ID_S, k > 0);
                }
                mma_commit(s_full + 8 * slot);
                mma_commit(k_empty + 8 * (n & 1));
            } else {
                bar_arrive(k_empty + 8 * (n & 1));
            }
        };
        uint32_t done = 0;                                                         // tiles done
        ok = __all_sync(0xffffffffu, wait(k_full, 0));
        fence_after();
        if (leader && ok) scores(0);
#pragma unroll 1
        for (int n = 0; n < n1 && ok; n++) {
            // the next keys are waited for before this tile's weights, so that S follows O at once
            const int st = n & 1;
            ok = wait(v_full + 8 * st, (n >> 1) & 1) && (n + 1 == n1 || wait(k_full + 8 * (st ^ 1), ((n + 1) >> 1) & 1)) &&
                 (!works(n) || wait(p_full + 8 * slot, done & 1));
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            if (leader) {
                if (works(n)) {
                    const uint64_t vd = v_desc + st * (M::TILE >> 4);
#pragma unroll
                    for (int k = 0; k < TC_TN / 16; k++)
                        mma_ts(o_tm, s_tm + 8 * k, vd + k * (2048 >> 4), ID_O, done > 0 || k > 0);
                    mma_commit(v_empty + 8 * st);
                } else {
                    bar_arrive(v_empty + 8 * st);
                }
                if (n + 1 < n1) scores(n + 1);
            }
            __syncwarp();
            done += works(n);
        }
        // the slot's output; nothing of this warp is in flight when the block ends, whatever ended the loop
        if (leader) {
            mma_commit(o_full + 8 * slot);
            for (int i = 0; i < 1 << 20 && !mbar_done(o_full + 8 * slot, 0); i++) {
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (wid == 15) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

int attend_error_flag(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_attend_error, sizeof(int)) != cudaSuccess) return -1;
    if (clear && v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_attend_error, &zero, sizeof(int));
    }
    return v ? 1 : 0;
}

int attend_tc_supported(int D, int dtype) { return (D == 64 || D == 128) && (dtype == KUSH_F16 || dtype == KUSH_BF16); }

template <int D, int BITS, int P, class IN, bool HELD>
static int launch_tc(const AttendArgs& a, int64_t tiles, cudaStream_t stream) {
    auto kern = attend_tc_kernel<D, BITS, P, IN, HELD>;
    constexpr int smem = TcSmem<D>::BYTES;
    static std::atomic<unsigned long long> attr_set{0};                            // one bit per device: the attribute is per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(attr_set.load() >> (dev & 63) & 1ull)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return set_error(KUSH_ERR_CUDA, "attention: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
        attr_set |= 1ull << (dev & 63);
    }
    launch_pdl(kern, dim3(unsigned(tiles), a.H, a.n_splits), dim3(TC_THREADS), size_t(smem), stream, a);
    return check_launch("attention (tensor cores)");
}

int launch_attend_tc(int D, int bits, int P, int dtype, const AttendArgs& a, int64_t rows, cudaStream_t stream) {
    const int64_t tiles = (rows * a.G + TC_TM - 1) / TC_TM + a.S;                  // at most one more per sequence
    if (tiles > 0x7fffffff || a.H > 65535 || a.n_splits > 65535)
        return set_error(KUSH_ERR_ARG, "attention: %lld row tiles, %d kv heads, %d splits", (long long)tiles, a.H, a.n_splits);
    if (a.held.limit_ms > 0) {
        if (D != 128 || bits != 4 || P != 16 || dtype != KUSH_BF16) return KUSH_ERR_UNSUPPORTED;
        return launch_tc<128, 4, 16, __nv_bfloat16, true>(a, tiles, stream);
    }
    return dispatch_fmt(D, bits, P, dtype, [&](auto Dc, auto Bc, auto Pc, auto in) -> int {
        using IN = decltype(in);
        if constexpr (Dc.value == 256 || std::is_same_v<IN, float>) return KUSH_ERR_UNSUPPORTED;
        else return launch_tc<Dc.value, Bc.value, Pc.value, IN, false>(a, tiles, stream);
    });
}

}  // namespace kush
