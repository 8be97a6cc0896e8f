// Paged attention for many query rows per kv head (prompts, chunks of prompts):
// bound by the tensor cores and the exponentials, so the products run on
// tcgen05 with the scores, weights and outputs in tensor memory.
//
// One persistent CTA per SM; an item is 256 rows (tokens x group heads) of one
// kv head as two 128-row tiles, so that a key tile (128 keys) read once serves both and
// one tile's softmax runs under the other's products. Warps:
//   0-3, 4-7  softmax of row tile 0 and 1: a thread owns a row;
//   8-11      load queries, keys and values into shared memory;
//   12        one thread issues the products (13-15 idle).
// Tensor memory (512 columns): S0, S1 (128 fp32 columns each), O0, O1 (D each).
// The weights P overwrite the first half of their S as 16-bit pairs and are the A
// operand of O += P V straight from tensor memory. Per row tile i and key tile j the
// issuing thread runs  O_i += P_i(j) V(j), S_i = Q_i K(j+1)^T  in that order: products
// of one thread execute in order, so S_i(j+1) cannot overtake the reading of P_i(j), and
// when its completion reaches the softmax warps, O_i is complete up to j and idle:
// they may rescale it without a barrier of its own. They do so only when a row's
// maximum grows by more than 2^8 (weights then stay below 2^8, exact in the sums).
//
// Shared memory holds operand rows of 64 elements (128 bytes) in the 128-byte
// swizzle: 16-byte chunk c of row r at chunk c ^ (r % 8). Queries and keys are K-major
// operands; values, stored key by key as they lie in the cache, are an MN-major B.
// The loaders write them with 16-byte cp.async, so any page size and any strides work;
// a 4-bit cache is widened to fp16 by the loaders (queries go to fp16 too, each
// row divided by a power of two), and the products see one type.
//
// Every wait is bounded: where one runs out, the CTA flags KVX_DEV_PIPE_TIMEOUT,
// all warps leave their loops, and tensor memory is freed.

#include <atomic>
#include <climits>
#include <type_traits>

#include "kvx.h"
#include "kvx_attn.cuh"
#include "kvx_host.h"

namespace kvx {

constexpr int kTileThreads = 512;
constexpr int kTileKeys = 128;
constexpr int kHalfRows = 128;                 // rows of one of the two row tiles
constexpr uint32_t kMaxWaitPolls = 1u << 22;   // each poll may suspend for a hardware-chosen time
constexpr int kLag = 2;                        // loads in flight before the oldest is awaited

template <int D>
struct TileConfig {
    static constexpr int kSlabs = D / 64;
    static constexpr int kSlabBytes = 128 * 128;                  // 128 rows of 64 elements
    static constexpr int kTileBytes = kSlabs * kSlabBytes;        // 128 rows of D elements
    static constexpr int kStages = D == 128 ? 5 : 8;              // ring of key and value tiles
    static constexpr int kRing = 2 * kTileBytes;                  // after the two query tiles
    static constexpr int kFactors = kRing + kStages * kTileBytes;
    static constexpr int kBars = kFactors + 2 * kHalfRows * 4;
    static constexpr int kSmem = 1024 + kBars + 256;
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
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
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

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
    const int n = take ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int R>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

template <int D>
struct TileBars {
    uint64_t full[TileConfig<D>::kStages], empty[TileConfig<D>::kStages];
    uint64_t q_full, q_empty;
    uint64_t s_full[2], p_full[2], o_full[2];
    uint64_t drain;
    uint32_t tmem;
    uint32_t abort;
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

__device__ __forceinline__ AttnItem tile_item(const AttnParams& p, int x) {
    const int per_slot = p.kv_heads * p.splits;
    const int slot = x / per_slot, rest = x - slot * per_slot;
    // The last tokens of a prompt see the most keys: their items go first.
    AttnItem it = locate_item(p, p.tile_slots - 1 - slot);
    it.head = rest / p.splits;
    it.split = rest - it.head * p.splits;
    return it;
}

template <typename T, int D, bool Q4>
__global__ void __launch_bounds__(kTileThreads, 1) attn_tile_kernel(const __grid_constant__ AttnParams p) {
    using C = TileConfig<D>;
    using M = typename std::conditional<Q4, __half, T>::type;       // type of the products' operands
    extern __shared__ char raw[];
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    char* smem = raw + (base - smem_addr(raw));
    float* factors = reinterpret_cast<float*>(smem + C::kFactors);  // what each query row was divided by
    auto* bars = reinterpret_cast<TileBars<D>*>(smem + C::kBars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_launch_dependents();
    if (warp == 12) {
        tmem_alloc(&bars->tmem, 512);
        if (lane == 0) {
            for (int i = 0; i < C::kStages; ++i) {
                mbar_init(&bars->full[i], 128);
                mbar_init(&bars->empty[i], 1);
            }
            mbar_init(&bars->q_full, 128);
            mbar_init(&bars->q_empty, 1);
            for (int i = 0; i < 2; ++i) {
                mbar_init(&bars->s_full[i], 1);
                mbar_init(&bars->p_full[i], 128);
                mbar_init(&bars->o_full[i], 1);
            }
            mbar_init(&bars->drain, 1);
            bars->abort = 0;
            mbar_init_fence();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    const uint32_t tmem = bars->tmem;
    uint32_t* abort = &bars->abort;
    const int items = p.tile_slots * p.kv_heads * p.splits;

    if (warp >= 12) {
        give_registers<40>();
        if (warp == 12 && lane == 0) {
            // ---- products ----
            constexpr uint32_t qk = instruction(std::is_same<M, __nv_bfloat16>::value, false, kTileKeys);
            constexpr uint32_t pv = instruction(std::is_same<M, __nv_bfloat16>::value, true, D);
            Ring<C::kStages> ring;
            uint32_t q_phase = 0, p_phase = 0;
            auto scores = [&](int i, int stage) {
                const uint32_t a = base + i * C::kTileBytes, b = base + C::kRing + stage * C::kTileBytes;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k / 4) * C::kSlabBytes + (k % 4) * 32;
                    tc_mma_ss(tmem + i * kTileKeys, operand(a + off, 16), operand(b + off, 16), qk, k > 0);
                }
                tc_commit(&bars->s_full[i]);
            };
            for (int x = blockIdx.x; x < items; x += gridDim.x) {
                const AttnItem it = tile_item(p, x);
                const KeyTiles kt = key_tiles<kTileKeys>(p, it);
                const int n = kt.end - kt.begin;
                if (n <= 0) continue;
                if (!bar_wait(&bars->q_full, q_phase, abort, p.status)) break;
                q_phase ^= 1;
                if (!bar_wait(&bars->full[ring.at], ring.phase, abort, p.status)) break;
                tc_fence_after();
                scores(0, ring.at);
                scores(1, ring.at);
                tc_commit(&bars->empty[ring.at]);
                ring.next();
                bool ok = true;
                for (int j = 0; j < n && ok; ++j) {
                    const Ring<C::kStages> v = ring;
                    ring.next();
                    if (!(ok = bar_wait(&bars->full[v.at], v.phase, abort, p.status))) break;
                    for (int i = 0; i < 2 && ok; ++i) {
                        if (!(ok = bar_wait(&bars->p_full[i], p_phase, abort, p.status))) break;
                        tc_fence_after();
                        const uint32_t b = base + C::kRing + v.at * C::kTileBytes;
#pragma unroll
                        for (int k = 0; k < kTileKeys / 16; ++k)
                            tc_mma_ts(tmem + 256 + i * D, tmem + i * kTileKeys + k * 8,
                                      operand(b + k * 2048, C::kSlabBytes), pv, j > 0 || k > 0);
                        if (j + 1 < n) {
                            if (i == 0) {
                                if (!(ok = bar_wait(&bars->full[ring.at], ring.phase, abort, p.status))) break;
                                tc_fence_after();
                            }
                            scores(i, ring.at);
                        } else {
                            tc_commit(&bars->o_full[i]);
                        }
                    }
                    if (!ok) break;
                    p_phase ^= 1;
                    tc_commit(&bars->empty[v.at]);
                    if (j + 1 < n) {
                        tc_commit(&bars->empty[ring.at]);
                        ring.next();
                    }
                }
                if (!ok) break;
                tc_commit(&bars->q_empty);
            }
            // Nothing of this CTA is in flight when its tensor memory is freed.
            tc_commit(&bars->drain);
            uint32_t never = 0;
            bar_wait(&bars->drain, 0, &never, p.status);
        }
        __syncwarp();
    } else if (warp >= 8) {
        give_registers<88>();
        // ---- loads ----
        const int w = warp - 8;
        Ring<C::kStages> ring;
        uint32_t q_phase = 1;                                       // the first query tile is free
        constexpr int kChunks = D / 8;                              // 16-byte chunks of a row of 16-bit elements
        constexpr int kRowsPerStep = 32 / kChunks;
        // Byte address of chunk c of row r in a tile of 128 rows.
        auto chunk_at = [](uint32_t tile, int r, int c) {
            return tile + (c >> 3) * C::kSlabBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        };
        if constexpr (!Q4) {
            uint64_t* pending[kLag] = {};
            int waiting = 0;                                        // loads issued and not yet announced
            bool ok = true;
            auto announce_oldest = [&]() {
                fence_async_shared();
                mbar_arrive(pending[0]);
#pragma unroll
                for (int i = 0; i + 1 < kLag; ++i) pending[i] = pending[i + 1];
                --waiting;
            };
            auto issued = [&](uint64_t* bar) {
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (waiting == kLag) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
                    announce_oldest();
                }
#pragma unroll
                for (int i = 0; i < kLag; ++i)
                    if (i == waiting) pending[i] = bar;
                ++waiting;
            };
            for (int x = blockIdx.x; x < items && ok; x += gridDim.x) {
                const AttnItem it = tile_item(p, x);
                const KeyTiles kt = key_tiles<kTileKeys>(p, it);
                const int n = kt.end - kt.begin;
                if (n <= 0) continue;
                const int last = it.pos0 + it.tokens - 1;
                const int32_t* table = p.table + it.seq * p.table_stride;
                const int64_t head_off = it.head * p.head_stride;
                const int q_after = n > 1 ? 3 : 2;                  // the queries follow this many key and value tiles
                for (int op = 0; op <= 2 * n; ++op) {
                    if (op == q_after) {
                        if (!(ok = warp_wait(&bars->q_empty, q_phase, abort, p.status))) break;
                        q_phase ^= 1;
                        int64_t off[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = 64 * w + 32 * h + lane, token = r / p.group;
                            off[h] = token < it.tokens ? (it.q0 + token) * p.q_token_stride +
                                                             (it.head * p.group + r - token * p.group) * p.q_head_stride
                                                       : -1;
                        }
#pragma unroll 4
                        for (int s = 0; s < 64; s += kRowsPerStep) {
                            const int r = s + lane / kChunks, c = lane % kChunks;
                            const int64_t a = __shfl_sync(~0u, s < 32 ? off[0] : off[1], r & 31);
                            const int row = 64 * w + r;
                            cp16(chunk_at(base + (row >> 7) * C::kTileBytes, row & 127, c), p.q + (a < 0 ? 0 : a) + 16 * c,
                                 a >= 0);
                        }
                        issued(&bars->q_full);
                    }
                    if (op == 2 * n) break;
                    if (!(ok = warp_wait(&bars->empty[ring.at], ring.phase ^ 1, abort, p.status))) break;
                    const int first = kt.first_key<kTileKeys>(kt.begin + (op >> 1));
                    const char* plane = (op & 1 ? p.v : p.k);
                    const uint32_t tile = base + C::kRing + ring.at * C::kTileBytes;
                    int64_t off = -1;
                    const int j = first + 32 * w + lane;
                    if (j <= last && (it.pos0 - j < p.window || j < p.sinks)) {
                        const int blk = block_of(p, j);
                        off = page_offset(p, table, blk);
                        if (off >= 0) off += (j - blk * p.block_size) * p.slot_stride + head_off;
                    }
#pragma unroll 4
                    for (int s = 0; s < 32; s += kRowsPerStep) {
                        const int r = s + lane / kChunks, c = lane % kChunks;
                        const int64_t a = __shfl_sync(~0u, off, r);
                        cp16(chunk_at(tile, 32 * w + r, c), plane + (a < 0 ? 0 : a) + 16 * c, a >= 0);
                    }
                    issued(&bars->full[ring.at]);
                    ring.next();
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (ok)
                while (waiting > 0) announce_oldest();
        } else {
            bool ok = true;
            for (int x = blockIdx.x; x < items && ok; x += gridDim.x) {
                const AttnItem it = tile_item(p, x);
                const KeyTiles kt = key_tiles<kTileKeys>(p, it);
                const int n = kt.end - kt.begin;
                if (n <= 0) continue;
                const int last = it.pos0 + it.tokens - 1;
                const int32_t* table = p.table + it.seq * p.table_stride;
                const int64_t head_off = it.head * p.head_stride;
                const int scales_at = p.block_size * (D / 2);
                const int q_after = n > 1 ? 3 : 2;
                const int t = lane & 3;                             // quarter of a row: D/4 elements
                constexpr int kWords = D / 32;                      // of codes a lane holds per key
                // A lane's codes and scales of four keys (8 apart) of a tile.
                uint32_t codes[4][kWords], scale[4];
                auto fetch = [&](int op) {
                    const int first = kt.first_key<kTileKeys>(kt.begin + (op >> 1)) + 32 * w;
                    const char* plane = (op & 1 ? p.v : p.k);
                    int64_t page = -1;
                    int off = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // block_size is a multiple of 16: 16 keys from a multiple of 16 share a page.
                        const int first16 = first + (i >> 1) * 16;
                        if ((i & 1) == 0) {
                            page = -1;
                            if (first16 <= last && (it.pos0 - (first16 + 15) < p.window || first16 < p.sinks)) {
                                const int blk = block_of(p, first16);
                                page = page_offset(p, table, blk);
                                off = first16 - blk * p.block_size;
                            }
                        }
                        const int key = (i & 1) * 8 + (lane >> 2), j = first16 + key;
                        scale[i] = 0;
#pragma unroll
                        for (int k = 0; k < kWords; ++k) codes[i][k] = 0;
                        if (page >= 0 && j <= last && (it.pos0 - j < p.window || j < p.sinks)) {
                            const char* b = plane + page + head_off;
                            const char* c = b + (off + key) * (D / 2) + t * (D / 8);
                            const char* s = b + scales_at + (off + key) * (D / 16);
                            if constexpr (D == 128) {
                                const uint4 v = __ldg(reinterpret_cast<const uint4*>(c));
                                codes[i][0] = v.x, codes[i][1] = v.y, codes[i][2] = v.z, codes[i][3] = v.w;
                                scale[i] = __ldg(reinterpret_cast<const uint16_t*>(s) + t);
                            } else {
                                const uint2 v = __ldg(reinterpret_cast<const uint2*>(c));
                                codes[i][0] = v.x, codes[i][1] = v.y;
                                scale[i] = __ldg(reinterpret_cast<const uint8_t*>(s) + t);
                            }
                        }
                    }
                };
                fetch(0);
                for (int op = 0; op <= 2 * n; ++op) {
                    if (op == q_after) {
                        if (!(ok = warp_wait(&bars->q_empty, q_phase, abort, p.status))) break;
                        q_phase ^= 1;
#pragma unroll 2
                        for (int s = 0; s < 64; s += kRowsPerStep) {
                            const int row = 64 * w + s + lane / kChunks, c = lane % kChunks;
                            const int token = row / p.group;
                            uint4 v = make_uint4(0, 0, 0, 0);
                            if (token < it.tokens)
                                v = *reinterpret_cast<const uint4*>(
                                    p.q + (it.q0 + token) * p.q_token_stride +
                                    (it.head * p.group + row - token * p.group) * p.q_head_stride + 16 * c);
                            float factor = 1.f;
                            if constexpr (!std::is_same<T, __half>::value) {
                                const float2 a = Pair<T>::unpack(v.x), b = Pair<T>::unpack(v.y), d = Pair<T>::unpack(v.z),
                                             e = Pair<T>::unpack(v.w);
                                float amax = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))),
                                                   fmaxf(fmaxf(fabsf(d.x), fabsf(d.y)), fmaxf(fabsf(e.x), fabsf(e.y))));
#pragma unroll
                                for (int k = 1; k < kChunks; k <<= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, k));
                                factor = row_divisor(amax);
                                const float inv = 1.f / factor;
                                v.x = Pair<__half>::pack(a.x * inv, a.y * inv);
                                v.y = Pair<__half>::pack(b.x * inv, b.y * inv);
                                v.z = Pair<__half>::pack(d.x * inv, d.y * inv);
                                v.w = Pair<__half>::pack(e.x * inv, e.y * inv);
                            }
                            st_shared16(chunk_at(base + (row >> 7) * C::kTileBytes, row & 127, c), v.x, v.y, v.z, v.w);
                            if (c == 0) factors[row] = factor;
                        }
                        fence_async_shared();
                        mbar_arrive(&bars->q_full);
                    }
                    if (op == 2 * n) break;
                    uint32_t now[4][kWords], now_scale[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        now_scale[i] = scale[i];
#pragma unroll
                        for (int k = 0; k < kWords; ++k) now[i][k] = codes[i][k];
                    }
                    if (op + 1 < 2 * n) fetch(op + 1);
                    if (!(ok = warp_wait(&bars->empty[ring.at], ring.phase ^ 1, abort, p.status))) break;
                    const uint32_t tile = base + C::kRing + ring.at * C::kTileBytes;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = 32 * w + 8 * i + (lane >> 2);
                        const uint32_t lo = now_scale[i] & 0xff, hi = D == 128 ? now_scale[i] >> 8 : lo;
                        const uint32_t s2[2] = {scales_to_half(lo | (lo << 8)), scales_to_half(hi | (hi << 8))};
#pragma unroll
                        for (int k = 0; k < kWords; ++k) {
                            uint32_t h[4];
                            codes_to_half(now[i][k], h);
                            const uint32_t s = s2[D == 128 ? k / 2 : 0];
                            st_shared16(chunk_at(tile, row, t * kWords + k), mul_half2(h[0], s), mul_half2(h[1], s),
                                        mul_half2(h[2], s), mul_half2(h[3], s));
                        }
                    }
                    fence_async_shared();
                    mbar_arrive(&bars->full[ring.at]);
                    ring.next();
                }
            }
        }
    } else {
        take_registers<192>();
        // ---- softmax ----
        const int i = warp >> 2;                                    // row tile
        const int row = (threadIdx.x & 127) + i * kHalfRows;        // row of the item
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + i * kTileKeys, o_at = tmem + lanes + 256 + i * D;
        const int token = row / p.group;
        const int head = row - token * p.group;
        uint32_t s_phase = 0, q_phase = 0, o_phase = 0;
        for (int x = blockIdx.x; x < items; x += gridDim.x) {
            const AttnItem it = tile_item(p, x);
            if (it.tokens == 0) continue;
            const KeyTiles kt = key_tiles<kTileKeys>(p, it);
            const int n = kt.end - kt.begin;
            const bool live = token < it.tokens;
            const int pos = live ? it.pos0 + token : -1;
            const int last = it.pos0 + it.tokens - 1;
            float top = -INFINITY, sum = 0.f;                       // raw score, sum of weights
            float scale = p.scale_log2;
            bool ok = true;
            if constexpr (Q4) {
                if (n > 0) {
                    if (!warp_wait(&bars->q_full, q_phase, abort, p.status)) break;
                    q_phase ^= 1;
                    scale *= factors[row];
                }
            }
            for (int j = 0; j < n; ++j) {
                if (!(ok = warp_wait(&bars->s_full[i], s_phase, abort, p.status))) break;
                s_phase ^= 1;
                tc_fence_after();
                uint32_t sr[kTileKeys];
#pragma unroll
                for (int c = 0; c < kTileKeys; c += 32) tmem_load32(s_at + c, sr + c);
                tc_wait_ld(sr);
#pragma unroll
                for (int c = 32; c < kTileKeys; c += 32) after_wait_ld(sr + c);
                const int first = kt.first_key<kTileKeys>(kt.begin + j);
                const bool whole = first + kTileKeys - 1 <= it.pos0 &&
                                   (last - first < p.window || first + kTileKeys - 1 < p.sinks);
                if (!whole) {
                    // Visible columns: [lo, hi] and those below `head_cols` (sinks).
                    const int hi = pos - first;
                    const int lo = pos - first >= p.window ? pos - first - p.window + 1 : 0;
                    const int head_cols = p.sinks - first;
#pragma unroll
                    for (int c = 0; c < kTileKeys; ++c)
                        if (c > hi || (c < lo && c >= head_cols)) sr[c] = __float_as_uint(-INFINITY);
                }
                float next = top;
#pragma unroll
                for (int c = 0; c < kTileKeys; ++c) next = fmaxf(next, __uint_as_float(sr[c]));
                // Keep the old maximum while weights stay below 2^8.
                const bool grow = j == 0 || (next - top) * scale > 8.f || top == -INFINITY;
                const float old = top;
                if (grow) top = next;
                const float ref = top == -INFINITY ? 0.f : top * scale;
                if (j > 0 && __any_sync(~0u, grow && next > old)) {
                    const float shrink = old == -INFINITY ? 0.f : exp2_approx(old * scale - ref);
                    sum *= shrink;
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_load32(o_at + c, o);
                        tc_wait_ld(o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
                        tmem_store32(o_at + c, o);
                    }
                }
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < kTileKeys; c += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float a = exp2_approx(fmaf(__uint_as_float(sr[c + k]), scale, -ref));
                        const float b = exp2_approx(fmaf(__uint_as_float(sr[c + k + 1]), scale, -ref));
                        part[k & 2] += a;
                        part[(k & 2) + 1] += b;
                        w[k / 2] = Pair<M>::pack(a, b);
                    }
                    tmem_store16(s_at + c / 2, w);
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&bars->p_full[i]);
            }
            if (!ok) break;
            if (n > 0) {
                if (!warp_wait(&bars->o_full[i], o_phase, abort, p.status)) break;
                o_phase ^= 1;
                tc_fence_after();
            }
            // A row that saw no key: sum 0.
            const float m2 = top == -INFINITY ? 0.f : top * scale;
            const float inv = p.out_scale / sum;
            const int64_t at = (static_cast<int64_t>(it.q0 + token) * p.heads + it.head * p.group + head) * p.splits + it.split;
            char* dst = p.out + (it.q0 + token) * p.o_token_stride + (it.head * p.group + head) * p.o_head_stride;
            if (live && p.splits > 1)
                *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(top == -INFINITY ? top : m2, sum);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float v[32];
                __syncwarp();
                if (n > 0) {
                    uint32_t o[32];
                    tmem_load32(o_at + c, o);
                    tc_wait_ld(o);
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(o[k]);
                }
                if (!live) continue;
                bool nan = false;
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    if (n <= 0 || sum == 0.f) v[k] = 0.f;
                    nan |= isnan(v[k]);
                }
                if (nan && !isnan(sum)) visible_keys_only<T, D, Q4, 32>(p, it, kt, kTileKeys, row, m2, c, v);
                if (p.splits > 1) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<float4*>(p.ws_o + at * D + c + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        uint32_t o[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            o[u] = sum == 0.f ? 0u : Pair<T>::pack(v[k + 2 * u] * inv, v[k + 2 * u + 1] * inv);
                        *reinterpret_cast<uint4*>(dst + (c + k) * 2) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            // O has been read: this thread's next arrival at p_full lets the products write it again.
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_free(tmem, 512);
}

template <typename T, int D, bool Q4>
static int run_tile(const AttnParams& p, int device, int sms, cudaStream_t stream) {
    constexpr int smem = TileConfig<D>::kSmem;
    static_assert(smem <= 227 * 1024 && sizeof(TileBars<D>) <= 256, "shared memory of the tile kernel");
    static std::atomic<uint64_t> done{0};               // devices that have the opt-in
    const uint64_t bit = 1ull << device;
    if (!(done.load(std::memory_order_relaxed) & bit)) {
        KVX_CUDA(cudaFuncSetAttribute(attn_tile_kernel<T, D, Q4>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                 "set attention kernel shared memory");
        // The roles' register shares add up to what 512 threads of 128 are launched with.
        cudaFuncAttributes attrs;
        KVX_CUDA(cudaFuncGetAttributes(&attrs, attn_tile_kernel<T, D, Q4>), "query attention kernel");
        if (attrs.numRegs != 128) return fail(KVX_EUNSUPPORTED, "attention kernel was built with %d registers", attrs.numRegs);
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    const int64_t items = static_cast<int64_t>(p.tile_slots) * p.kv_heads * p.splits;
    if (items > INT_MAX) return fail(KVX_EUNSUPPORTED, "too many tiles of queries for one call");
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
    KVX_CUDA(cudaLaunchKernelEx(&cfg, attn_tile_kernel<T, D, Q4>, p), "launch attention kernel");
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
