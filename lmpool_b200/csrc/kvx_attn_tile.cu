// Paged attention for many query rows per kv head (prompts, chunks of prompts):
// bound by the tensor cores and the exponentials, so the products run on
// tcgen05 with the scores, weights and outputs in tensor memory.
//
// One persistent CTA per SM; an item is 256 rows (tokens x group heads) of one
// kv head as two 128-row tiles, so that a key tile (128 keys) read once serves both and
// one tile's softmax runs under the other's products. Warps:
//   0-3, 4-7  softmax of row tile 0 and 1: a thread owns a row;
//   8-11      queries into shared memory; edge tiles of a 16-bit cache; widening of a 4-bit one;
//   12, 15    issue the products of row tile 0 and 1 (two warps, because a wait of one stands in
//             the queue behind its own products: one warp for both left the tensor cores idle
//             half of the time);
//   13        issues the bulk copies;
//   14        looks up items ahead (lengths, offsets, ranges of keys);
//   16-19     write finished rows while the others are at the next item.
// Tensor memory (512 columns): per row tile two score buffers of 64 columns (S), then
// O0, O1 (D each). A step is 64 keys: S_i(u) = Q_i K(u)^T into buffer u % 2; its weights P
// overwrite the first half of the buffer as 16-bit pairs and are the A operand of O_i +=
// P_i(u) V(u) straight from tensor memory. The issuing warp runs, per step,
// O_i += P_i(u) V(u), then S_i(u + 2) into the buffer that this frees: the softmax of step
// u + 1 has its scores already and never waits for a product of its own. (With one
// buffer of 128 keys it did, for the 1400 clocks of both products: 3300 clocks per 128 keys.)
// Products of one thread execute in order, so S_i(u + 2) cannot overtake the reading of P_i(u).
// A row's maximum may be stale by 2^8 (weights stay below 2^8, 2^15 in fp16: kLift; exact in the sums); only
// when it grows by more do the softmax warps rescale O, once O_i += P_i(u - 1) is done.
//
// Shared memory holds operand rows of 64 elements (128 bytes) in the 128-byte
// swizzle: 16-byte chunk c of row r at chunk c ^ (r % 8). Queries and keys are K-major
// operands; values, stored key by key as they lie in the cache, are an MN-major B.
// A 16-bit cache whose page size is a multiple of 8 is read by TMA, one box per page (or 128 rows
// of it) and 64 elements. The value tile that reaches behind the context, and every tile of a
// cache of other page sizes, is gathered by 16-byte cp.async instead, with zeros for
// keys that no row sees: what lies behind a context may be NaN, and 0 * NaN is not 0.
// A 4-bit cache comes as raw pages through a ring of its own (bulk copies of 16 keys or more) and
// is widened to fp16 in shared memory (queries go to fp16 too, each row divided by a power of
// two), so that the products see one type.
//
// Exponentials: the special-function unit gives 16 a clock and SM, which alone is as
// long as the products of a tile. So some are computed as 2^n p(f), x = n + f, |f| <=
// 1/2, on the FMA units, with a degree-4 polynomial (relative error 2.8e-6, from a
// weighted least-squares fit of 2^f; the weights are rounded to 2^-8 or 2^-11).
//
// Measured: a prompt of 8191 tokens, window 1024, 32 query heads on 8: 201 us (76 us of products at the rate of a large
// library product); 4 prompts of 129 to 4095 tokens on up to 2001 earlier ones: 438 us (218 us); two of 3001 to 4096 on a
// 4-bit cache: 380 us (183 us). Counters of a prompt of 4096 tokens: tensor cores 48 % of the time busy, issue slots 51 %, ALU
// 34 %, special-function units 30 %, no unit full; warps wait (most for tensor memory and barriers): what bounds it is the chain of
// a step, scores to softmax to weights to product, of which two row tiles run at a time. Instructions in the softmax loop stand
// in that chain: two more values kept in it, 4 %.
//
// Every wait is bounded: where one runs out, the CTA flags KVX_DEV_PIPE_TIMEOUT,
// all warps leave their loops, and tensor memory is freed.

#include <cuda.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "kvx.h"
#include "kvx_attn.cuh"
#include "kvx_host.h"

namespace kvx {

constexpr int kTileThreads = 640;
constexpr int kTileKeys = 128;
constexpr int kStepKeys = 64;                  // keys of a step
constexpr int kHalfRows = 128;                 // rows of one of the two row tiles
// Of 8 pairs of exponentials, on the FMA units: 3 on a 16-bit cache (8 prompts of 2048: 319 us, 322 with none), 1
// on a 4-bit one, where the widening wants the issue slots (two prompts on a 4-bit cache: 389 us, 407 with 3).
template <bool Q4>
constexpr int kFmaPairs = Q4 ? 1 : 3;
constexpr float kFarScore = 1 << 20;           // log2 of a weight's factor is off by at most 2^-4 below this
constexpr uint32_t kMaxWaitPolls = 1u << 22;   // each poll may suspend for a hardware-chosen time

template <int D, bool Q4>
struct TileConfig {
    static constexpr int kSlabs = D / 64;
    static constexpr int kSlabBytes = 128 * 128;                  // 128 rows of 64 elements
    static constexpr int kTileBytes = kSlabs * kSlabBytes;        // 128 rows of D elements
    static constexpr int kStages = D == 128 ? (Q4 ? 4 : 5) : 8;   // ring of key and value tiles
    static constexpr int kRawStages = Q4 ? 3 : 0;                 // ring of raw 4-bit tiles
    static constexpr int kRawCodes = kTileKeys * D / 2;
    static constexpr int kRawBytes = kRawCodes + kTileKeys * D / 16;
    static constexpr int kRing = 2 * kTileBytes;                  // after the two query tiles
    static constexpr int kRaw = kRing + kStages * kTileBytes;
    static constexpr int kFactors = kRaw + kRawStages * kRawBytes;
    static constexpr int kSums = kFactors + (Q4 ? 2 * kHalfRows * 4 : 0);
    static constexpr int kBars = kSums + 2 * kHalfRows * 4;
    static constexpr int kSmem = 1024 + kBars + 768;
};

// TMA views of a 16-bit cache: [D, block_size, kv_heads, num_blocks] from the innermost.
struct TileMaps {
    CUtensorMap k, v;
    int32_t box_rows;      // rows of a box; 0: no TMA
};

// ---- tcgen05 ----------------------------------------------------------------

__device__ __forceinline__ void tmem_alloc(uint32_t* at, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The registers of earlier tensor-memory loads are valid from here on: named as operands, so that no use moves up.
#define KVX_REGS32(r)                                                                                                   \
    "+r"((r)[0]), "+r"((r)[1]), "+r"((r)[2]), "+r"((r)[3]), "+r"((r)[4]), "+r"((r)[5]), "+r"((r)[6]), "+r"((r)[7]),      \
        "+r"((r)[8]), "+r"((r)[9]), "+r"((r)[10]), "+r"((r)[11]), "+r"((r)[12]), "+r"((r)[13]), "+r"((r)[14]),           \
        "+r"((r)[15]), "+r"((r)[16]), "+r"((r)[17]), "+r"((r)[18]), "+r"((r)[19]), "+r"((r)[20]), "+r"((r)[21]),         \
        "+r"((r)[22]), "+r"((r)[23]), "+r"((r)[24]), "+r"((r)[25]), "+r"((r)[26]), "+r"((r)[27]), "+r"((r)[28]),         \
        "+r"((r)[29]), "+r"((r)[30]), "+r"((r)[31])
__device__ __forceinline__ void tc_wait_ld(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : KVX_REGS32(r)::"memory");
}
__device__ __forceinline__ void after_wait_ld(uint32_t* r) { asm volatile("" : KVX_REGS32(r)::"memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// Arrives at `bar` when every product issued so far by this thread is done.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
// D (tensor memory) = A B (+ D); A in shared memory or in tensor memory.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// 32 lanes (of this warp's quarter) x 32 columns, one row a thread.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::
                       "memory");
}
__device__ __forceinline__ void tmem_load8(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// Shared-memory operand descriptor: 128-byte swizzle, groups of 8 rows 1024 bytes
// apart; `lead` is the distance of 64-element slabs (MN-major operands only).
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fff) | (static_cast<uint64_t>(lead >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: fp32 accumulators, 16-bit operands of one type, M = 128.
__host__ __device__ constexpr uint32_t instruction(bool bf16, bool mn_major_b, int n) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (mn_major_b ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n / 8) << 17) | (static_cast<uint32_t>(128 / 16) << 24);
}

__device__ __forceinline__ void st_shared16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int block,
                                          uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(slot), "r"(head), "r"(block), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void raw_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

// Two floats in one register pair.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// The largest of three; NaN where one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The n lowest bits; none for n <= 0, all for n >= 32.
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}
// 32 bytes of one row: a whole memory sector where the address allows it.
__device__ __forceinline__ void store32(void* p, const uint32_t* r, bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                     "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(r[0], r[1], r[2], r[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(r[4], r[5], r[6], r[7]);
    }
}
// 2^x on the FMA units for x <= 127: x = n + f by adding and taking away 1.5 * 2^23 (n then
// stands in the low bits), 2^f as a polynomial with p(0) = 1, and n added to its exponent.
// What is below -127 becomes exactly 0: p(0) 2^-127 has an empty exponent and fraction.
__device__ __forceinline__ uint64_t exp2_fma(uint64_t x) {
    const float2 v = unpair(x);
    x = pair2(fmaxf(v.x, -127.f), fmaxf(v.y, -127.f));
    const uint64_t r = add2(x, pair2(12582912.f, 12582912.f));
    const uint64_t f = fma2(add2(r, pair2(-12582912.f, -12582912.f)), pair2(-1.f, -1.f), x);
    uint64_t y = fma2(f, pair2(0.009582853f, 0.009582853f), pair2(0.055906426f, 0.055906426f));
    y = fma2(y, f, pair2(0.240240991f, 0.240240991f));
    y = fma2(y, f, pair2(0.693124175f, 0.693124175f));
    y = fma2(y, f, pair2(1.f, 1.f));
    const float2 n = unpair(r), m = unpair(y);
    return pair2(__uint_as_float(__float_as_uint(n.x) * 0x800000u + __float_as_uint(m.x)),
                 __uint_as_float(__float_as_uint(n.y) * 0x800000u + __float_as_uint(m.y)));
}

template <int R>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

// An item with its keys, as warp 14 hands it to the others.
struct TileWork {
    AttnItem it;
    KeyTiles kt;
};
constexpr int kWork = 4;       // items looked up ahead
constexpr int kRoles = 19;     // warps that take each item: all but 14

template <int D, bool Q4>
struct TileBars {
    uint64_t full[TileConfig<D, Q4>::kStages], empty[TileConfig<D, Q4>::kStages];
    uint64_t raw_full[4], raw_empty[4];
    uint64_t q_full, q_empty;
    uint64_t s_full[2][2], p_full[2][2];     // [row tile][score buffer]
    uint64_t pv_done[2], o_full[2], o_free[2], sums_full[2];
    uint64_t drain, idle;
    uint64_t work_full[kWork], work_empty[kWork];
    TileWork work[kWork];
    uint32_t raw_bad[4];       // 16-key groups of a raw tile that were not copied
    uint32_t tmem;
    uint32_t abort;
    uint32_t spoiled;          // rows that warps 16-19 are to look over again
};

// Waits for the barrier's phase; false when another warp gave up or the polls ran out.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, uint32_t* abort, int32_t* status) {
    for (uint32_t i = 0; i < kMaxWaitPolls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*reinterpret_cast<volatile uint32_t*>(abort)) return false;
    }
    *reinterpret_cast<volatile uint32_t*>(abort) = 1;
    atomicOr(status, KVX_DEV_PIPE_TIMEOUT);
    return false;
}

// The same for a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* abort, int32_t* status) {
    return __all_sync(~0u, bar_wait(bar, parity, abort, status));
}

// A position in a ring of N barriers.
template <int N>
struct Ring {
    int at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) at = 0, phase ^= 1;
    }
};

// The items of a call, without gaps, as one warp walks them: tiles of queries from the last sequence's
// last to the first (the last tokens of a prompt see the most keys: they go first), and of
// each every kv head and split. Sequences are counted 32 at a time, one a lane; the walk only
// goes on, so that it passes over them once.
struct ItemWalk {
    int chunk;      // sequences 32 * chunk ... are in view
    int after;      // tiles of the sequences behind them
    int tiles;      // this lane's sequence: its tiles
    int upto;       // and those of the lanes from here on
    int all;        // tiles of the 32

    __device__ __forceinline__ int tiles_of(const AttnParams& p, int s, bool report) const {
        if (s >= p.num_seqs) return 0;
        if (p.cu == nullptr) return 1;
        const int a = p.cu[s], b = p.cu[s + 1];
        if (a < 0 || b < a || b > p.num_tokens) {
            if (report) atomicOr(p.status, KVX_DEV_BAD_LEN);
            return 0;
        }
        return (b - a + p.tile_tokens - 1) / p.tile_tokens;
    }
    __device__ __forceinline__ void view(const AttnParams& p, int c) {
        const int lane = threadIdx.x & 31;
        chunk = c;
        tiles = tiles_of(p, 32 * c + lane, false);
        upto = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int other = __shfl_down_sync(~0u, upto, d);
            if (lane + d < 32) upto += other;
        }
        all = __shfl_sync(~0u, upto, 0);
    }
    // Starts the walk; the number of tiles of the call.
    __device__ __forceinline__ int64_t start(const AttnParams& p) {
        int64_t n = 0;
        for (int s = threadIdx.x & 31; s < p.num_seqs; s += 32) n += tiles_of(p, s, true);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(~0u, n, d);
        after = 0;
        view(p, (p.num_seqs - 1) / 32);
        return n;
    }
    // Tile y (counted from the end), not before an earlier call's.
    __device__ __forceinline__ AttnItem tile(const AttnParams& p, int y) {
        while (y >= after + all && chunk > 0) {
            after += all;
            view(p, chunk - 1);
        }
        const int rest = y - after;                                  // in this chunk, from its end
        const uint32_t hit = __ballot_sync(~0u, rest < upto && rest >= upto - tiles);
        const int who = hit ? __ffs(hit) - 1 : 0;
        const int tile = __shfl_sync(~0u, upto - 1 - rest, who);     // of its sequence, from its start
        AttnItem it;
        it.seq = 32 * chunk + who;
        it.head = it.split = 0;
        const int a = p.cu ? p.cu[it.seq] : it.seq, len = p.cu ? p.cu[it.seq + 1] - a : 1;
        const int first = tile * p.tile_tokens;
        it.q0 = a + first;
        it.tokens = hit ? min(p.tile_tokens, len - first) : 0;
        it.pos0 = context_of(p, it.seq) - len + first;
        return it;
    }
};

// Item x of the call (kv heads and splits of a tile of queries follow each other: `per_tile` of them).
__device__ __forceinline__ void item_of(const AttnParams& p, ItemWalk& walk, int64_t x, int per_tile, TileWork& w) {
    const int y = static_cast<int>(x / per_tile), rest = static_cast<int>(x - static_cast<int64_t>(y) * per_tile);
    w.it = walk.tile(p, y);
    w.it.head = rest / p.splits;
    w.it.split = rest - w.it.head * p.splits;
    w.kt = key_tiles<kTileKeys>(p, w.it);
}

// Marks the NaN elements of an output row whose sum is a number, by the thread that wrote it, and notes in `spoiled` that
// there are some (there may be where `dst` is null: partial results).
template <typename T, int D>
__device__ __noinline__ void mark_row(char* dst, volatile uint32_t* spoiled) {
    uint16_t* out = reinterpret_cast<uint16_t*>(dst);
    bool any = dst == nullptr;
    for (int d = 0; d < D && dst != nullptr; ++d)
        if ((out[d] & 0x7fff) > Pair<T>::kInf) {
            out[d] = marked_nan<T>();
            any = true;
        }
    if (any) *spoiled = 1;
}

// The rows that one of warps 16-19 wrote, looked over once more when the CTA's items are done (see mend_row): nobody
// waits for this warp then, so that no input can make a wait run out.
template <typename T, int D, bool Q4>
__device__ __noinline__ void mend_items(const AttnParams& p) {
    ItemWalk walk;
    const int per_tile = p.kv_heads * p.splits;
    const int64_t items = walk.start(p) * per_tile;
    const int base = (threadIdx.x & 127) & ~31;
    int hint = -1;
    for (int64_t x = blockIdx.x; x < items; x += gridDim.x) {
        TileWork w;
        item_of(p, walk, x, per_tile, w);
        if (w.kt.begin == w.kt.end) continue;
        for (int r = 0; r < 64; ++r) {
            const int row = (r >> 5) * kHalfRows + base + (r & 31), token = row / p.group;
            if (token >= w.it.tokens) continue;
            if (p.splits > 1) {
                const int head = w.it.head * p.group + row - token * p.group;
                const int64_t at = (static_cast<int64_t>(w.it.q0 + token) * p.heads + head) * p.splits + w.it.split;
                if (isnan(p.ws_ml[at * 2 + 1])) continue;           // its scores: nothing to mend
            }
            mend_row<T, D, Q4>(p, w.it, w.kt, kTileKeys, row, true, &hint);
        }
    }
}

// Whether an item has rows in its second row tile.
__device__ __forceinline__ bool second_tile(const AttnParams& p, const AttnItem& it) { return it.tokens * p.group > kHalfRows; }

// Whether a tile of a 16-bit cache is gathered row by row: always without TMA, else the value
// tile (odd op) that reaches behind the context.
__device__ __forceinline__ bool gathered(int box_rows, int op, int first, int last) {
    return box_rows == 0 || ((op & 1) && first + kTileKeys - 1 > last);
}

// The copies of one CTA, by one warp: TMA boxes of a 16-bit cache into the operand
// ring, raw pages of a 4-bit cache into the ring of raw tiles. A lane looks up one box or run
// of 16 keys and copies it, so that a tile's page lookups are in flight together.
template <int D, bool Q4>
__device__ __forceinline__ void issue_copies(const AttnParams& p, const TileMaps& maps, uint32_t base, TileBars<D, Q4>* bars) {
    using C = TileConfig<D, Q4>;
    Ring<Q4 ? C::kRawStages : C::kStages> ring;
    uint32_t* abort = &bars->abort;
    const int lane = threadIdx.x & 31;
    const int run = Q4 ? 16 : maps.box_rows;            // keys of a copy
    const int at = lane * run;                          // this lane's first key in a tile
    Ring<kWork> work;
    while (true) {
        AttnItem it;
        KeyTiles kt;
        if (!take_work(bars, work, p.status, it, kt)) return;
        const int n = kt.end - kt.begin;
        const int last = it.pos0 + it.tokens - 1;
        const int32_t* table = p.table + it.seq * p.table_stride;
        // This lane's page of a tile, if some row sees its keys. On a 4-bit cache it is read while the tile before is copied
        // (8 prompts of 2048, fp16: 363 us, 384 if read before the wait for its place in the ring, 371 after it; bf16: 389, 385
        // and 394).
        bool wanted = false;
        int id = -1, slot = 0;
        auto look_up = [&](int tile) {
            const int j = kt.first_key<kTileKeys>(kt.begin + tile) + at;
            wanted = run > 0 && tile < n && at < kTileKeys && j <= last && (it.pos0 - (j + run - 1) < p.window || j < p.sinks);
            id = -1;
            if (wanted) {
                const int blk = block_of(p, j);
                slot = j - blk * p.block_size;
                if (blk < p.table_width) id = table[blk];
            }
        };
        if (Q4) look_up(0);
        for (int op = 0; op < 2 * n; ++op, ring.next()) {
            if constexpr (!Q4) {
                if (!warp_wait(&bars->empty[ring.at], ring.phase ^ 1, abort, p.status)) return;
                if (run == 0 || gathered(run, op, kt.first_key<kTileKeys>(kt.begin + (op >> 1)), last)) {
                    if (lane == 0) mbar_arrive(&bars->full[ring.at]);
                    continue;
                }
                if (!(op & 1)) look_up(op >> 1);
            }
            if constexpr (Q4)
                if (!warp_wait(&bars->raw_empty[ring.at], ring.phase ^ 1, abort, p.status)) return;
            if (wanted && (id < 0 || id >= p.num_blocks)) {
                atomicOr(p.status, KVX_DEV_BAD_SRC_ID);
                id = -1;
            }
            if constexpr (!Q4) {
                uint64_t* bar = &bars->full[ring.at];
                if (lane == 0) mbar_arrive_expect_tx(bar, C::kTileBytes);
                __syncwarp();
                const uint32_t tile = base + C::kRing + ring.at * C::kTileBytes;
                // What is not to be read comes from outside the cache: zeros.
                if (at < kTileKeys)
#pragma unroll
                    for (int c = 0; c < C::kSlabs; ++c)
                        tma_load4(tile + c * C::kSlabBytes + at * 128, op & 1 ? &maps.v : &maps.k, 64 * c, slot, it.head,
                                  id < 0 ? static_cast<int>(p.num_blocks) : id, bar);
            } else {
                uint64_t* bar = &bars->raw_full[ring.at];
                const uint32_t take = __ballot_sync(~0u, id >= 0);
                if (lane == 0) {
                    *reinterpret_cast<volatile uint32_t*>(&bars->raw_bad[ring.at]) = ~take;
                    mbar_arrive_expect_tx(bar, __popc(take) * 16 * (D / 2 + D / 16));
                }
                __syncwarp();
                const uint32_t raw = base + C::kRaw + ring.at * C::kRawBytes;
                if (id >= 0) {
                    const char* src = (op & 1 ? p.v : p.k) + it.head * p.head_stride + id * p.block_stride;
                    raw_copy(raw + at * (D / 2), src + slot * (D / 2), 16 * (D / 2), bar);
                    raw_copy(raw + C::kRawCodes + at * (D / 16), src + p.block_size * (D / 2) + slot * (D / 16),
                             16 * (D / 16), bar);
                }
            }
            if (Q4 && (op & 1)) look_up((op >> 1) + 1);
        }
    }
}

// The next item of a role (a whole warp), copied out of the ring that warp 14 fills; false after the last
// one, or when the CTA gave up.
template <int D, bool Q4>
__device__ __forceinline__ bool take_work(TileBars<D, Q4>* bars, Ring<kWork>& ring, int32_t* status, AttnItem& it, KeyTiles& kt) {
    if (!warp_wait(&bars->work_full[ring.at], ring.phase, &bars->abort, status)) return false;
    it = bars->work[ring.at].it;
    kt = bars->work[ring.at].kt;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&bars->work_empty[ring.at]);
    ring.next();
    return it.seq >= 0;
}

template <typename T, int D, bool Q4>
__global__ void __launch_bounds__(kTileThreads, 1) attn_tile_kernel(const __grid_constant__ AttnParams p,
                                                                  const __grid_constant__ TileMaps maps) {
    using C = TileConfig<D, Q4>;
    using M = typename std::conditional<Q4, __half, T>::type;       // type of the products' operands
    extern __shared__ char raw[];
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    char* smem = raw + (base - smem_addr(raw));
    float* factors = reinterpret_cast<float*>(smem + C::kFactors);  // what each query row was divided by
    float* sums = reinterpret_cast<float*>(smem + C::kSums);        // sums of weights, for warps 16-19
    auto* bars = reinterpret_cast<TileBars<D, Q4>*>(smem + C::kBars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_launch_dependents();
    if (warp == 12) {
        tmem_alloc(&bars->tmem, 512);
        if (lane == 0) {
            for (int i = 0; i < C::kStages; ++i) {
                mbar_init(&bars->full[i], Q4 ? 128 : 5);    // 16-bit: warps 8-11 and 13
                mbar_init(&bars->empty[i], 2);
            }
            for (int i = 0; i < 4; ++i) {
                mbar_init(&bars->raw_full[i], 1);
                mbar_init(&bars->raw_empty[i], 128);
            }
            mbar_init(&bars->q_full, 128);
            mbar_init(&bars->q_empty, 2);
            for (int i = 0; i < 2; ++i) {
                for (int h = 0; h < 2; ++h) {
                    mbar_init(&bars->s_full[i][h], 1);
                    mbar_init(&bars->p_full[i][h], 128);
                }
                mbar_init(&bars->pv_done[i], 1);
                mbar_init(&bars->o_full[i], 1);
                mbar_init(&bars->o_free[i], 128);
                mbar_init(&bars->sums_full[i], 128);
            }
            mbar_init(&bars->drain, 2);
            mbar_init(&bars->idle, 128);
            for (int i = 0; i < kWork; ++i) {
                mbar_init(&bars->work_full[i], 1);
                mbar_init(&bars->work_empty[i], kRoles);
            }
            bars->abort = 0;
            bars->spoiled = 0;
            mbar_init_fence();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    constexpr uint32_t tmem = 0;               // all 512 columns are this CTA's: they start at 0
    uint32_t* abort = &bars->abort;

    // Registers: 5 x 96 a thread at launch; from here on 2 x 128, 72, 56, and 96 for the warps that call functions.
    if (warp >= 16) {
        // ---- finished rows ----
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        uint32_t phases[2] = {0, 0};
        bool ok = true;
        Ring<kWork> work;
        while (ok) {
            AttnItem it;
            KeyTiles kt;
            if (!take_work(bars, work, p.status, it, kt)) break;
            if (it.tokens == 0) continue;
            const int n = kt.end - kt.begin;
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
                if (i == 1 && !second_tile(p, it)) break;
                const uint32_t phase = i ? phases[1] : phases[0];
                const int row = (threadIdx.x & 127) + i * kHalfRows;
                const int token = row / p.group, head = row - token * p.group;
                const bool live = token < it.tokens;
                const uint32_t o_at = tmem + lanes + 256 + i * D;
                float sum = 0.f;
                if (n > 0) {
                    if (!(ok = warp_wait(&bars->sums_full[i], phase, abort, p.status))) break;
                    if (!(ok = warp_wait(&bars->o_full[i], phase, abort, p.status))) break;
                    tc_fence_after();
                    sum = sums[row];
                }
                // A row that saw no key has the sum 0 and gives zeros.
                const bool none = sum == 0.f;
                const float inv = none ? 0.f : p.out_scale / sum;
                const int64_t at =
                    (static_cast<int64_t>(it.q0 + token) * p.heads + it.head * p.group + head) * p.splits + it.split;
                char* dst = p.out + (it.q0 + token) * p.o_token_stride + (it.head * p.group + head) * p.o_head_stride;
                if (n <= 0 && p.splits > 1) {                       // a split without keys: the join reads no more of it
                    if (live) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(-INFINITY, 0.f);
                    continue;
                }
                bool nan = false;
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t o[16];
                    __syncwarp();
                    if (n > 0) tmem_load16(o_at + c, o);
                    if (none) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = 0;
                    }
                    float any = 0.f;                                // NaN where an element is not finite
#pragma unroll
                    for (int k = 0; k < 16; ++k) any = fmaf(__uint_as_float(o[k]), 0.f, any);
                    nan |= isnan(any);
                    if (!live) {
                    } else if (p.splits > 1) {
                        store32(p.ws_o + at * D + c, o, true);
                        store32(p.ws_o + at * D + c + 8, o + 8, true);
                    } else {
                        uint32_t h[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            h[u] = Pair<T>::pack(__uint_as_float(o[2 * u]) * inv, __uint_as_float(o[2 * u + 1]) * inv);
                        store32(dst + c * 2, h, p.out_wide);
                    }
                }
                if (n > 0) {
                    tc_fence_before();
                    mbar_arrive(&bars->o_free[i]);
                }
                if (live && nan && !isnan(sum)) mark_row<T, D>(p.splits > 1 ? nullptr : dst, &bars->spoiled);
            }
            if (n > 0) {
                phases[0] ^= 1;
                if (second_tile(p, it)) phases[1] ^= 1;
            }
        }
        __syncwarp();
        if (__any_sync(~0u, *reinterpret_cast<volatile uint32_t*>(&bars->spoiled))) mend_items<T, D, Q4>(p);
    } else if (warp >= 12) {
        give_registers<56>();
        if (warp == 12 || warp == 15) {
            // ---- products of one row tile ---- (the whole warp keeps step, one lane issues)
            const int i = warp == 15;
            constexpr uint32_t qk = instruction(std::is_same<M, __nv_bfloat16>::value, false, kStepKeys);
            constexpr uint32_t pv = instruction(std::is_same<M, __nv_bfloat16>::value, true, D);
            const bool leader = elect_one();
            const uint64_t q_desc = operand(base + i * C::kTileBytes, 16), k_desc = operand(base + C::kRing, 16),
                           v_desc = operand(base + C::kRing, C::kSlabBytes);
            const uint32_t s_at = tmem + i * 2 * kStepKeys, o_at = tmem + 256 + i * D;
            Ring<C::kStages> ring;
            Ring<kWork> work;
            uint32_t q_phase = 0, p_phase = 0, free_phase = 1;
            [[maybe_unused]] uint32_t idle_phase = 0;
            // Scores against the keys of half h of a stage, into buffer h.
            auto scores = [&](int h, int stage) {
                if (leader) {
                    const uint64_t b = k_desc + stage * (C::kTileBytes >> 4) + h * (kStepKeys * 128 >> 4);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const int off = ((k / 4) * C::kSlabBytes + (k % 4) * 32) >> 4;
                        tc_mma_ss(s_at + h * kStepKeys, q_desc + off, b + off, qk, k > 0);
                    }
                    tc_commit(&bars->s_full[i][h]);
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (leader) tc_commit(bar);
                __syncwarp();
            };
            while (true) {
                AttnItem it;
                KeyTiles kt;
                if (!take_work(bars, work, p.status, it, kt)) break;
                const int n = kt.end - kt.begin;
                if (n <= 0) continue;
                if (!warp_wait(&bars->q_full, q_phase, abort, p.status)) break;
                q_phase ^= 1;
                if (i == 1 && !second_tile(p, it)) {
                    // No rows here: the stages are let go as they come.
                    bool ok = true;
                    for (int op = 0; op < 2 * n; ++op, ring.next()) {
                        if (!(ok = warp_wait(&bars->full[ring.at], ring.phase, abort, p.status))) break;
                        if (lane == 0) mbar_arrive(&bars->empty[ring.at]);
                    }
                    if (ok && Q4) ok = warp_wait(&bars->idle, idle_phase, abort, p.status);
                    if (!ok) break;
                    idle_phase ^= 1;
                    if (lane == 0) mbar_arrive(&bars->q_empty);
                    continue;
                }
                if (!warp_wait(&bars->full[ring.at], ring.phase, abort, p.status)) break;
                tc_fence_after();
                scores(0, ring.at);
                scores(1, ring.at);
                commit(&bars->empty[ring.at]);
                ring.next();
                bool ok = true;
                for (int j = 0; j < n && ok; ++j) {
                    const Ring<C::kStages> v = ring;
                    ring.next();
                    if (!(ok = warp_wait(&bars->full[v.at], v.phase, abort, p.status))) break;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!(ok = warp_wait(&bars->p_full[i][h], p_phase, abort, p.status))) break;
                        if (j == 0 && h == 0 && !(ok = warp_wait(&bars->o_free[i], free_phase, abort, p.status))) break;
                        tc_fence_after();
                        if (leader) {
                            const uint64_t b = v_desc + v.at * (C::kTileBytes >> 4) + h * (kStepKeys * 128 >> 4);
#pragma unroll
                            for (int k = 0; k < kStepKeys / 16; ++k)
                                tc_mma_ts(o_at, s_at + h * kStepKeys + k * 8, b + k * (2048 >> 4), pv, j > 0 || h > 0 || k > 0);
                            tc_commit(&bars->pv_done[i]);
                        }
                        __syncwarp();
                        if (j + 1 == n) {
                            if (h == 1) commit(&bars->o_full[i]);
                            continue;
                        }
                        if (h == 0) {
                            if (!(ok = warp_wait(&bars->full[ring.at], ring.phase, abort, p.status))) break;
                            tc_fence_after();
                        }
                        scores(h, ring.at);
                    }
                    if (!ok) break;
                    p_phase ^= 1;
                    commit(&bars->empty[v.at]);
                    if (j + 1 < n) {
                        commit(&bars->empty[ring.at]);
                        ring.next();
                    }
                    // No product of this row tile reads these queries any more. (With a single key tile only now, when
                    // its softmax warps have shown that they are past the item's factors.)
                    if (j + 2 == n || n == 1) commit(&bars->q_empty);
                }
                if (!ok) break;
                free_phase ^= 1;
            }
            // Nothing of this CTA is in flight when its tensor memory is freed.
            commit(&bars->drain);
            uint32_t never = 0;
            bar_wait(&bars->drain, 0, &never, p.status);
        }
        __syncwarp();
        if (warp == 13) issue_copies<D, Q4>(p, maps, base, bars);
        if (warp == 14) {
            Ring<kWork> ring;
            ItemWalk walk;
            const int per_tile = p.kv_heads * p.splits;
            const int64_t items = walk.start(p) * per_tile;
            for (int64_t x = blockIdx.x;; x += gridDim.x, ring.next()) {
                TileWork next = {};
                next.it.seq = -1;                                    // no more items
                if (x < items) item_of(p, walk, x, per_tile, next);
                if (!warp_wait(&bars->work_empty[ring.at], ring.phase ^ 1, abort, p.status)) break;
                if (lane == 0) {
                    bars->work[ring.at] = next;
                    mbar_arrive(&bars->work_full[ring.at]);
                }
                if (next.it.seq < 0) break;
            }
        }
    } else if (warp >= 8) {
        give_registers<72>();
        // ---- queries, edge tiles, widening ----
        const int w = warp - 8;
        Ring<C::kStages> ring;
        Ring<Q4 ? C::kRawStages : 1> raw;
        uint32_t q_phase = 1;                                       // the first query tile is free
        constexpr int kChunks = D / 8;                              // 16-byte chunks of a row of 16-bit elements
        constexpr int kRowsPerStep = 32 / kChunks;
        // Byte address of chunk c of row r in a tile of 128 rows.
        auto chunk_at = [](uint32_t tile, int r, int c) {
            return tile + (c >> 3) * C::kSlabBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        };
        int my_token[2], my_head[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = kHalfRows * h + 32 * w + lane;
            my_token[h] = row / p.group;
            my_head[h] = row - my_token[h] * p.group;
        }
        bool ok = true, fresh = true;
        Ring<kWork> work;
        while (ok) {
            AttnItem it;
            KeyTiles kt;
            if (!take_work(bars, work, p.status, it, kt)) break;
            const int n = kt.end - kt.begin;
            if (n <= 0) continue;
            const int last = it.pos0 + it.tokens - 1;
            // The queries follow this many key and value tiles of the item. (The first item's come before them: nothing
            // is in their place yet, and no product can start without them.)
            const int q_after = fresh ? 0 : n > 1 ? 3 : 2;
            fresh = false;
            const int row_tiles = second_tile(p, it) ? 2 : 1;
            for (int op = 0; op <= 2 * n; ++op) {
                if (op == q_after) {
                    if (!(ok = warp_wait(&bars->q_empty, q_phase, abort, p.status))) break;
                    q_phase ^= 1;
                    int64_t off[2];                                 // of this lane's row of each row tile
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        off[h] = my_token[h] < it.tokens ? (it.q0 + my_token[h]) * p.q_token_stride +
                                                               (it.head * p.group + my_head[h]) * p.q_head_stride
                                                         : -1;
#pragma unroll 1
                    for (int h = 0; h < row_tiles; ++h) {
                        const int64_t mine = h ? off[1] : off[0];
#pragma unroll 4
                        for (int s = 0; s < 32; s += kRowsPerStep) {
                            const int r = s + lane / kChunks, c = lane % kChunks;
                            const int64_t from = __shfl_sync(~0u, mine, r);
                            cp_async16(chunk_at(base + h * C::kTileBytes, 32 * w + r, c), p.q + 16 * c + (from >= 0 ? from : 0), from >= 0);
                        }
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    if constexpr (Q4 && !std::is_same<T, __half>::value) {
                        // To fp16 in place, a lane a row: the largest magnitude first (bf16 bits without their sign are
                        // ordered as numbers), then the elements over its power of two.
                        __syncwarp();
#pragma unroll 1
                        for (int h = 0; h < row_tiles; ++h) {
                            const int row = kHalfRows * h + 32 * w + lane;
                            if (__all_sync(~0u, (h ? my_token[1] : my_token[0]) >= it.tokens)) {
                                factors[row] = 1.f;                 // no rows here: zeros already
                                continue;
                            }
                            const uint32_t tile = base + h * C::kTileBytes;
                            uint32_t big = 0;
#pragma unroll 4
                            for (int c = 0; c < kChunks; ++c) {
                                const uint4 v = ld_shared16(chunk_at(tile, row & 127, c));
                                big = max_u16x2(big, max_u16x2(max_u16x2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                                               max_u16x2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
                            }
                            const uint32_t most = max(big & 0xffffu, big >> 16);
                            const float factor = row_divisor(__uint_as_float(most << 16)), inv = 1.f / factor;
                            factors[row] = factor;
#pragma unroll 4
                            for (int c = 0; c < kChunks; ++c) {
                                const uint32_t at = chunk_at(tile, row & 127, c);
                                const uint4 v = ld_shared16(at);
                                const float2 a = Pair<T>::unpack(v.x), b = Pair<T>::unpack(v.y), d = Pair<T>::unpack(v.z),
                                             e = Pair<T>::unpack(v.w);
                                st_shared16(at, Pair<__half>::pack(a.x * inv, a.y * inv),
                                            Pair<__half>::pack(b.x * inv, b.y * inv), Pair<__half>::pack(d.x * inv, d.y * inv),
                                            Pair<__half>::pack(e.x * inv, e.y * inv));
                            }
                        }
                    } else if constexpr (Q4) {
                        for (int h = 0; h < 2; ++h) factors[kHalfRows * h + 32 * w + lane] = 1.f;
                    }
                    fence_async_shared();
                    mbar_arrive(&bars->q_full);
                }
                if (op == 2 * n) break;
                const int first = kt.first_key<kTileKeys>(kt.begin + (op >> 1));
                const uint32_t tile = base + C::kRing + ring.at * C::kTileBytes;
                if constexpr (!Q4) {
                    // Warp 13 and these four go through every stage together, whichever of them fills it: a
                    // barrier's phases are told apart by parity alone, so none may fall two behind.
                    if (!(ok = warp_wait(&bars->empty[ring.at], ring.phase ^ 1, abort, p.status))) break;
                    if (gathered(maps.box_rows, op, first, last)) {
                        int64_t off = -1;
                        const int j = first + 32 * w + lane;
                        if (j <= last && (it.pos0 - j < p.window || j < p.sinks)) {
                            const int blk = block_of(p, j);
                            off = page_offset(p, p.table + it.seq * p.table_stride, blk);
                            if (off >= 0) off += (j - blk * p.block_size) * p.slot_stride + it.head * p.head_stride;
                        }
                        const char* plane = op & 1 ? p.v : p.k;
#pragma unroll 4
                        for (int s = 0; s < 32; s += kRowsPerStep) {
                            const int r = s + lane / kChunks, c = lane % kChunks;
                            const int64_t a = __shfl_sync(~0u, off, r);
                            cp_async16(chunk_at(tile, 32 * w + r, c), plane + (a < 0 ? 0 : a) + 16 * c, a >= 0);
                        }
                        asm volatile("cp.async.wait_all;" ::: "memory");
                        fence_async_shared();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars->full[ring.at]);
                } else {
                    if (!(ok = warp_wait(&bars->raw_full[raw.at], raw.phase, abort, p.status))) break;
                    if (!(ok = warp_wait(&bars->empty[ring.at], ring.phase ^ 1, abort, p.status))) break;
                    const uint32_t from = base + C::kRaw + raw.at * C::kRawBytes;
                    const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&bars->raw_bad[raw.at]);
                    const int t = lane & 3;                         // quarter of a row: D/4 elements
                    constexpr int kWords = D / 32;                  // of codes a lane holds per key
                    // Every key of the tile is seen by some row and lies in a good page.
                    const bool all = (bad & 0xff) == 0 && first + kTileKeys - 1 <= last &&
                                     (it.pos0 - first < p.window || first + kTileKeys - 1 < p.sinks);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = 32 * w + 8 * i + (lane >> 2), j = first + row;
                        uint32_t codes[kWords], scale;
                        // The right half of the row's words comes first in lanes 2 and 3 of a row: the 16-byte
                        // stores of eight lanes then fall on eight different bank groups.
                        const int flip = D == 128 ? (t >> 1) * 2 : 0;
                        const uint32_t at = from + row * (D / 2) + t * (D / 8);
                        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(codes[0]), "=r"(codes[1]) : "r"(at + flip * 4));
                        if constexpr (D == 128) {
                            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                                         : "=r"(codes[2]), "=r"(codes[3])
                                         : "r"(at + (flip ^ 2) * 4));
                            uint16_t u;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(from + C::kRawCodes + row * 8 + t * 2));
                            scale = u;
                        } else {
                            uint16_t u;
                            asm volatile("ld.shared.u8 %0, [%1];" : "=h"(u) : "r"(from + C::kRawCodes + row * 4 + t));
                            scale = u;
                        }
                        // Keys that no row sees and bad pages read as zeros, whatever the raw tile holds.
                        if (!all && (((bad >> (row >> 4)) & 1) || j > last || (it.pos0 - j >= p.window && j >= p.sinks))) scale = 0;
                        const uint32_t lo = scale & 0xff, hi = D == 128 ? scale >> 8 : lo;
                        const uint32_t s_lo = scales_to_half(lo | (lo << 8)), s_hi = scales_to_half(hi | (hi << 8));
#pragma unroll
                        for (int k = 0; k < kWords; ++k) {
                            uint32_t h[4];
                            codes_to_half(codes[k], h);
                            const int word = k ^ flip;              // words 0, 1: first 16 elements, 2, 3: the others
                            const uint32_t s = D == 128 && (word & 2) ? s_hi : s_lo;
                            st_shared16(chunk_at(tile, row, t * kWords + word), mul_half2(h[0], s), mul_half2(h[1], s),
                                        mul_half2(h[2], s), mul_half2(h[3], s));
                        }
                    }
                    mbar_arrive(&bars->raw_empty[raw.at]);
                    raw.next();
                    fence_async_shared();
                    mbar_arrive(&bars->full[ring.at]);
                }
                ring.next();
            }
        }
        if constexpr (!Q4) asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        take_registers<128>();
        // ---- softmax ----
        const int i = warp >> 2;                                    // row tile
        const int row = (threadIdx.x & 127) + i * kHalfRows;        // row of the item
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + i * 2 * kStepKeys, o_at = tmem + lanes + 256 + i * D;
        const int token = row / p.group;
        const int head = row - token * p.group;
        [[maybe_unused]] uint32_t q_phase = 0;
        uint32_t s_phase = 0, free_phase = 1, pv_phase = 1;
        Ring<kWork> work;
        while (true) {
            AttnItem it;
            KeyTiles kt;
            if (!take_work(bars, work, p.status, it, kt)) break;
            const int n = kt.end - kt.begin;
            if (n <= 0) continue;
            const bool idle = i == 1 && !second_tile(p, it);
            [[maybe_unused]] float factor = 1.f;
            if constexpr (Q4) {
                // In idle items too, and acknowledged: a barrier's phases are told apart by parity alone, so the
                // queries of the next item must not come before these warps have seen those of this one.
                if (!warp_wait(&bars->q_full, q_phase, abort, p.status)) break;
                q_phase ^= 1;
                factor = factors[row];
                if (idle) mbar_arrive(&bars->idle);
            }
            if (idle) continue;
            const bool live = token < it.tokens;
            const int pos = live ? it.pos0 + token : -1;
            const int last = it.pos0 + it.tokens - 1;
            float top = -INFINITY, sum = 0.f;                       // raw score, sum of weights
            float scale = p.scale_log2;
            bool ok = true;
            if constexpr (Q4) scale *= factor;
#pragma unroll 1
            for (int u = 0; u < 2 * n; ++u) {
                const int h = u & 1;
                if (!(ok = warp_wait(&bars->s_full[i][h], s_phase, abort, p.status))) break;
                s_phase ^= h;
                tc_fence_after();
                const uint32_t at = s_at + h * kStepKeys;
                uint32_t sr[kStepKeys];
                tmem_load32(at, sr);
                tmem_load32(at + 32, sr + 32);
                const int first = kt.first_key<kTileKeys>(kt.begin + (u >> 1)) + h * kStepKeys;
                const bool whole = first + kStepKeys - 1 <= it.pos0 &&
                                   (last - first < p.window || first + kStepKeys - 1 < p.sinks);
                tc_wait_ld(sr);
                after_wait_ld(sr + 32);
                if (!whole) {
                    // Columns that this row sees, as bits: [lo, hi] and those below `head_cols` (sinks).
                    const int hi = pos - first;
                    const int lo = pos - first >= p.window ? pos - first - p.window + 1 : 0;
                    const int head_cols = p.sinks - first;
#pragma unroll
                    for (int b = 0; b < kStepKeys; b += 32) {
                        const uint32_t seen = low_bits(hi + 1 - b) & (~low_bits(lo - b) | low_bits(head_cols - b));
#pragma unroll
                        for (int c = 0; c < 32; ++c) sr[b + c] = seen & (1u << c) ? sr[b + c] : 0xff800000u;
                    }
                }
                // Four chains of three-way maxima; NaN where a score is NaN.
                float best[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kStepKeys; c += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        best[k] = max3(best[k], __uint_as_float(sr[c + 2 * k]), __uint_as_float(sr[c + 2 * k + 1]));
                const float next = max3(max3(best[0], best[1], best[2]), best[3], best[3]);
                // Keep the old maximum while weights stay below 2^8.
                const bool grow = u == 0 || (!(next == top) && !((next - top) * scale <= 8.f));
                const float old = top;
                if (grow) top = next;
                // A score that is infinite, itself or only when scaled, gives NaN, as inf - inf does in the formula.
                const float lead = top * scale;
                float ref = lead == -INFINITY ? 0.f : lead == INFINITY ? NAN : lead - kLift<M>;
                // Below, score * scale - ref is rounded once, so that the largest weight is off by 2 to the rounding of `lead`:
                // a factor that the sum has too, but one that must stay small. Rows of larger scores subtract first. (One
                // vote for both rare cases: with two, prompts take 2 % longer.)
                const bool far = fabsf(lead) >= kFarScore && lead != -INFINITY;
                if (__any_sync(~0u, grow || far)) {
                    if (u > 0 && __any_sync(~0u, grow)) {
                        const float shrink = !grow ? 1.f : old == -INFINITY ? 0.f : exp2_approx((old - top) * scale);
                        sum *= shrink;
                        if (!(ok = warp_wait(&bars->pv_done[i], pv_phase, abort, p.status))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 8) {
                            uint32_t o[8];
                            tmem_load8(o_at + c, o);
#pragma unroll
                            for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
                            tmem_store8(o_at + c, o);
                        }
                    }
                    if (__any_sync(~0u, far)) {
                        const float zero = top == -INFINITY ? 0.f : top;
                        ref = ref == ref ? -kLift<M> : ref;
#pragma unroll
                        for (int c = 0; c < kStepKeys; c += 2) {
                            const float2 d = unpair(add2(pair2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), pair2(-zero, -zero)));
                            sr[c] = __float_as_uint(d.x);
                            sr[c + 1] = __float_as_uint(d.y);
                        }
                    }
                }
                const uint64_t scale2 = pair2(scale, scale), ref2 = pair2(-ref, -ref);
                uint64_t part[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < kStepKeys; c += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const uint64_t e = fma2(pair2(__uint_as_float(sr[c + 2 * k]), __uint_as_float(sr[c + 2 * k + 1])),
                                                scale2, ref2);
                        uint64_t y;
                        if ((k & 7) < kFmaPairs<Q4>) {
                            y = exp2_fma(e);
                        } else {
                            const float2 v = unpair(e);
                            y = pair2(exp2_approx(v.x), exp2_approx(v.y));
                        }
                        part[k & 1] = add2(part[k & 1], y);
                        const float2 v = unpair(y);
                        w[k] = Pair<M>::pack(v.x, v.y);
                    }
                    tmem_store16(at + c / 2, w);
                }
                const float2 total = unpair(add2(part[0], part[1]));
                sum += total.x + total.y;
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&bars->p_full[i][h]);
                pv_phase ^= 1;                                      // of the product that these weights are for
            }
            if (!ok) break;
            if (live && p.splits > 1) {
                const int64_t at =
                    (static_cast<int64_t>(it.q0 + token) * p.heads + it.head * p.group + head) * p.splits + it.split;
                *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(top == -INFINITY ? top : top * scale - kLift<M>, sum);
            }
            // The row's sum goes to warps 16-19 when they are done with the item before.
            if (!warp_wait(&bars->o_free[i], free_phase, abort, p.status)) break;
            free_phase ^= 1;
            sums[row] = sum;
            mbar_arrive(&bars->sums_full[i]);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // After a wait that ran out, copies may still be on their way into this CTA's shared memory: 1 ms is
    // a thousand times what one takes.
    if (*reinterpret_cast<volatile uint32_t*>(abort))
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    if (warp == 12) tmem_free(bars->tmem, 512);
}

// cuTensorMapEncodeTiled, from the driver that is loaded.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int encode_maps(const AttnParams& p, int head_dim, bool bf16, TileMaps* maps) {
    maps->box_rows = 0;
    int rows = p.block_size & -p.block_size;            // the largest power of two that divides a page
    if (rows < 8) return KVX_OK;                        // the swizzle repeats every 8 rows
    rows = rows > kTileKeys ? kTileKeys : rows;
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p.slot_stride), static_cast<cuuint64_t>(p.head_stride),
                                   static_cast<cuuint64_t>(p.block_stride)};
    for (const cuuint64_t st : strides)
        if (st == 0 || st >= (1ull << 40)) return KVX_OK;     // also negative ones
    if (p.num_blocks > 0x7fffffff) return KVX_OK;
    static std::atomic<EncodeTiled> encode{nullptr};
    EncodeTiled fn = encode.load(std::memory_order_acquire);
    if (fn == nullptr) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult found;
        KVX_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &sym, 12000, cudaEnableDefault, &found),
                 "find cuTensorMapEncodeTiled");
        if (sym == nullptr) return fail(KVX_ECUDA, "cuTensorMapEncodeTiled not available from the driver");
        fn = reinterpret_cast<EncodeTiled>(sym);
        encode.store(fn, std::memory_order_release);
    }
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(p.block_size),
                                static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.num_blocks)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1}, steps[4] = {1, 1, 1, 1};
    for (int i = 0; i < 2; ++i) {
        const CUresult r = fn(i ? &maps->v : &maps->k,
                              bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                              const_cast<char*>(i ? p.v : p.k), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return KVX_OK;           // a layout that TMA does not take is gathered
    }
    maps->box_rows = rows;
    return KVX_OK;
}

template <typename T, int D, bool Q4>
static int run_tile(const AttnParams& p, int device, int sms, cudaStream_t stream) {
    constexpr int smem = TileConfig<D, Q4>::kSmem;
    static_assert(smem <= 227 * 1024 && sizeof(TileBars<D, Q4>) <= 768, "shared memory of the tile kernel");
    static std::atomic<uint64_t> done{0};               // devices that have the opt-in
    const uint64_t bit = 1ull << device;
    if (!(done.load(std::memory_order_relaxed) & bit)) {
        KVX_CUDA(cudaFuncSetAttribute(attn_tile_kernel<T, D, Q4>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                 "set attention kernel shared memory");
        // The roles' register shares add up to at most what 640 threads of 96 are launched with.
        cudaFuncAttributes attrs;
        KVX_CUDA(cudaFuncGetAttributes(&attrs, attn_tile_kernel<T, D, Q4>), "query attention kernel");
        if (attrs.numRegs != 96) return fail(KVX_EUNSUPPORTED, "attention kernel was built with %d registers", attrs.numRegs);
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    const int64_t items = static_cast<int64_t>(p.tile_slots) * p.kv_heads * p.splits;
    if (items > INT_MAX) return fail(KVX_EUNSUPPORTED, "too many tiles of queries for one call");
    TileMaps maps = {};
    if (!Q4) {
        const int rc = encode_maps(p, D, std::is_same<T, __nv_bfloat16>::value, &maps);
        if (rc != KVX_OK) return rc;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items < sms ? items : sms));
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    KVX_CUDA(cudaLaunchKernelEx(&cfg, attn_tile_kernel<T, D, Q4>, p, maps), "launch attention kernel");
    return KVX_OK;
}

int launch_attn_tile(const AttnParams& p, int head_dim, int dtype, bool q4, int device, int sms, cudaStream_t stream) {
    const auto run = head_dim == 64 ? (q4 ? (dtype ? run_tile<__half, 64, true> : run_tile<__nv_bfloat16, 64, true>)
                                          : (dtype ? run_tile<__half, 64, false> : run_tile<__nv_bfloat16, 64, false>))
                                    : (q4 ? (dtype ? run_tile<__half, 128, true> : run_tile<__nv_bfloat16, 128, true>)
                                          : (dtype ? run_tile<__half, 128, false> : run_tile<__nv_bfloat16, 128, false>));
    return run(p, device, sms, stream);
}

}  // namespace kvx
