// Paged attention for few query rows per kv head (decode, drafted tokens):
// bound by the bytes of the cache, so every warp streams its own keys and the
// work is split over the key axis until the GPU is full.
//
// An item is up to 8 * NT rows (tokens x group heads) of one kv head and one
// range of 64-key tiles; its four warps take 16 keys of a tile each and keep
// their own running maximum and sum, so the loop has no barrier among warps. Keys are
// the M side of the products: S^T = K Q^T and O^T = V^T P^T with m16n8k16, so
// that the usual 4 to 8 rows of a group fill an n = 8 tile (rows on the M side
// would leave half or more of every product empty).
//
// 16-bit cache: each warp has a ring of kStages slices (16 keys of K and V) in
// shared memory, filled by 16-byte cp.async (any page size, any strides; keys
// that no row sees are filled with zeros), read back by ldmatrix.
// 4-bit cache: the ring holds raw slices (16 keys: 1 KiB of codes and 128 bytes of scales of K
// and of V at head_dim 128, each contiguous in a page), which lanes widen to fp16 and scale on
// their way into the products, exactly. The fragments' order along head_dim and along the keys
// is free as long as both operands agree, so a lane takes the codes that lie together. A slice takes a warp about 450
// instructions, half of them the widening (eight for eight elements with the scaling, and V's masks and shifts); with four warps a
// scheduler the issue slots are 60 % busy and the ALU 51 %: half of what bounds this path is the latency between them, not
// the bytes. Queries go to fp16 too, each row first divided by the power of two below its
// largest element.
// Measured, bf16, head_dim 128: 4 sequences of 40000 to 65610 keys, 4 rows of 8 kv heads: 139 us, 6.1 TB/s, 0.95
// of the copy rate; 256 of 500 to 4095 keys, window 1024, 8 rows: 174 us, 0.92. 4-bit: 64 sequences of 1000 to 8191 keys,
// 4 rows: 97 us, 0.53 of the copy rate; one of 131070 keys, 8 rows: 48 us, 0.48. A call of a few sequences takes
// 11 us, of which the launch and the host's call are most.
// Weights: for a bf16 cache they are split in two bf16 numbers (2^-17 relative;
// the tensor cores have time to spare here), for fp16 and 4-bit rounded to fp16, 2^7 higher (kLift).

#include <atomic>
#include <climits>
#include <type_traits>

#include "kvx.h"
#include "kvx_attn.cuh"
#include "kvx_host.h"

namespace kvx {

constexpr int kSplitWarps = 4;
constexpr int kQ4Slices = 2;
constexpr int kQ4Stages = 2;

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <typename T>
__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int N>
__device__ __forceinline__ void ld_shared(uint32_t (&r)[N], uint32_t addr) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
    else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t addr) {
    uint32_t r;
    asm volatile("{\n\t.reg .u16 t;\n\tld.shared.u16 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(r) : "r"(addr) : "memory");
    return r;
}
__device__ __forceinline__ uint32_t ld_shared_u8(uint32_t addr) {
    uint32_t r;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
    return r;
}

template <int D, int NT, bool Q4>
struct SplitConfig {
    static constexpr int kSlices = Q4 && NT < 3 ? kQ4Slices : 1;             // slices of 16 keys a warp takes at once
    static constexpr int kWarpKeys = 16 * kSlices;
    static constexpr int kKeys = kWarpKeys * kSplitWarps;                    // keys of a tile
    static constexpr int kStages = Q4 ? kQ4Stages : 3;
    static constexpr int kCodes = 16 * D / 2, kScales = 16 * D / 16;         // bytes of a 4-bit slice, K or V
    static constexpr int kStageBytes = Q4 ? kSlices * 2 * (kCodes + kScales) : 2 * 16 * D * 2;
    static constexpr int kRing = kStages * kStageBytes * kSplitWarps;
    static constexpr int kMerge = kSplitWarps * 8 * NT * (D + 4) * 4;
    static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

template <typename T, int D, int NT, bool Q4>
__global__ void __launch_bounds__(kSplitWarps * 32, Q4 && NT == 1 ? 4 : 2) attn_split_kernel(const __grid_constant__ AttnParams p) {
    using M = typename std::conditional<Q4, __half, T>::type;     // type of the products' operands
    using C = SplitConfig<D, NT, Q4>;
    constexpr int kRows = 8 * NT;
    constexpr int KS = D / 16;                                     // k steps of Q K^T, m tiles of V^T P^T
    constexpr int NS = C::kSlices;
    constexpr bool kTwoWeights = !Q4 && std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(128) char smem[];
    griddep_launch_dependents();
    griddep_wait();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    // Every sequence is looked at by one thread of the call (there are at least num_seqs slots).
    if (p.cu != nullptr && threadIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && blockIdx.x < p.num_seqs)
        check_offsets(p, blockIdx.x);
    AttnItem it = locate_item(p, blockIdx.x);
    it.head = blockIdx.y;
    it.split = blockIdx.z;
    if (it.tokens == 0) return;
    const KeyTiles kt = key_tiles<C::kKeys>(p, it);
    const int rows = it.tokens * p.group;
    if (kt.begin == kt.end && p.splits > 1) {                      // a split without keys: the join reads no more of it
        for (int row = threadIdx.x; row < rows; row += kSplitWarps * 32) {
            const int64_t at = (static_cast<int64_t>(it.q0 + row / p.group) * p.heads + it.head * p.group + row % p.group) *
                                   p.splits + it.split;
            *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(-INFINITY, 0.f);
        }
        return;
    }
    const int32_t* table = p.table + it.seq * p.table_stride;
    const int last = it.pos0 + it.tokens - 1;
    const int64_t head_off = it.head * p.head_stride;
    [[maybe_unused]] const char* k_head = p.k + head_off;
    [[maybe_unused]] const char* v_head = p.v + head_off;

    // Whether any row of the item sees key j: what no row sees counts nowhere.
    auto wanted = [&](int j) { return j <= last && (it.pos0 - j < p.window || j < p.sinks); };
    // Whether a slice of 16 keys holds such a key; whether all of them are.
    auto touched = [&](int first) { return first <= last && (it.pos0 - (first + 15) < p.window || first < p.sinks); };
    auto filled = [&](int first) { return first + 15 <= last && (it.pos0 - first < p.window || first + 15 < p.sinks); };
    auto first_of = [&](int i, int sub) { return kt.template first_key<C::kKeys>(i) + warp * C::kWarpKeys + 16 * sub; };

    // Where this warp's slices lie, for pages that hold whole slices: a lane looks up one of the next 32
    // slices, a batch ahead, so that no load of keys waits for a table entry.
    const bool paged16 = p.block_size % 16 == 0;
    int64_t run_now = -1, run_next = -1;                           // bytes from the head's first key in page 0
    int gap_now = 0, gap_next = 0;                                 // 4-bit: from the slice's codes to its scales
    auto look_up = [&](int batch) {
        const int m = batch * 32 + lane, i = kt.begin + m / NS;
        run_next = -1;
        if (i < kt.end) {
            const int first = first_of(i, m % NS);
            if (touched(first)) {
                const int blk = block_of(p, first), in = first - blk * p.block_size;
                run_next = page_offset(p, table, blk);
                if (run_next >= 0) run_next += in * (Q4 ? D / 2 : p.slot_stride);
                gap_next = p.block_size * (D / 2) - in * (D / 2 - D / 16);
            }
        }
    };
    auto advance = [&](int n) {                                    // before the slices of iteration n are read
        if ((n * NS) % 32 == 0) {
            run_now = run_next;
            gap_now = gap_next;
            look_up(n * NS / 32 + 1);
        }
    };
    const int count = kt.end - kt.begin;
    if (paged16) look_up(0);

    // 16-bit cache: slice n of this warp into a stage of its ring.
    [[maybe_unused]] const uint32_t ring = smem_addr(smem) + warp * C::kStages * C::kStageBytes;
    [[maybe_unused]] auto fetch16 = [&](int n, int stage) {
        if (n < count) {
            constexpr int kChunks = D / 8;                         // 16-byte chunks of a row
            constexpr int kRowsPerStep = 32 / kChunks;
            const int first = first_of(kt.begin + n, 0);
            const int c = lane % kChunks, r_lane = lane / kChunks;
            const uint32_t dst = ring + stage * C::kStageBytes;
            int64_t off = -1;                                      // of this lane's row
            bool all = false;
            if (paged16) {
                advance(n);
                const int64_t run = __shfl_sync(~0u, run_now, n & 31);
                all = filled(first) && run >= 0;
                off = run < 0 ? -1 : run + head_off + r_lane * p.slot_stride;
            } else {
                const int j = first + (lane & 15);
                if (wanted(j)) {
                    const int blk = block_of(p, j);
                    off = page_offset(p, table, blk);
                    if (off >= 0) off += (j - blk * p.block_size) * p.slot_stride + head_off;
                }
            }
            if (all) {
                const char* k_src = p.k + off + 16 * c;
                const char* v_src = p.v + off + 16 * c;
#pragma unroll
                for (int r0 = 0; r0 < 16; r0 += kRowsPerStep) {
                    const int r = r0 + r_lane;
                    const uint32_t to = dst + r * (D * 2) + ((c ^ (r & 7)) << 4);
                    cp_async16(to, k_src + r0 * p.slot_stride, true);
                    cp_async16(to + 16 * D * 2, v_src + r0 * p.slot_stride, true);
                }
            } else {
                // Zeros for keys that no row sees and for bad pages.
#pragma unroll
                for (int r0 = 0; r0 < 16; r0 += kRowsPerStep) {
                    const int r = r0 + r_lane;
                    int64_t a = paged16 ? off + r0 * p.slot_stride : __shfl_sync(~0u, off, r);
                    if (paged16 && (off < 0 || !wanted(first + r))) a = -1;
                    const int64_t from = (a < 0 ? 0 : a) + c * 16;
                    const uint32_t to = dst + r * (D * 2) + ((c ^ (r & 7)) << 4);
                    cp_async16(to, p.k + from, a >= 0);
                    cp_async16(to + 16 * D * 2, p.v + from, a >= 0);
                }
            }
        }
        cp_async_commit();
    };
    // 4-bit cache: the slices of iteration n into a stage. block_size is a multiple of 16. Keys are
    // rows of the products in the order 0 4 1 5 2 6 3 7 (and 8 further): a lane's four keys
    // of V are then t, t + 4, t + 8 and t + 12, rows side by side. Key k of K stands at the
    // row it is; V's 16-byte chunks are crossed in every second pair of rows, against bank conflicts.
    constexpr int kRowChunks = D / 32;                             // 16-byte chunks of a row of codes
    [[maybe_unused]] auto fetch4 = [&](int n, int stage) {
        if (n < count) {
            advance(n);
#pragma unroll
            for (int z = 0; z < NS; ++z) {
                const int64_t run = __shfl_sync(~0u, run_now, (n * NS + z) & 31);
                const int gap = __shfl_sync(~0u, gap_now, (n * NS + z) & 31);
                const bool take = run >= 0;                        // else nothing to see or a bad page: zeros
                const char* k_from = k_head + (take ? run : 0);
                const char* v_from = v_head + (take ? run : 0);
                const uint32_t dst = ring + stage * C::kStageBytes + z * 2 * (C::kCodes + C::kScales);
#pragma unroll
                for (int h = 0; h < C::kCodes / 512; ++h) {
                    const int chunk = lane + 32 * h, key = chunk / kRowChunks, c = chunk % kRowChunks;
                    const int k_row = (key & 8) | ((key & 3) << 1) | ((key >> 2) & 1);
                    cp_async16(dst + k_row * (D / 2) + c * 16, k_from + chunk * 16, take);
                    cp_async16(dst + C::kCodes + key * (D / 2) + (c ^ (D == 128 ? key & 2 : 0)) * 16, v_from + chunk * 16, take);
                }
                constexpr int kScaleChunks = C::kScales / 16;
                if (lane < 2 * kScaleChunks)
                    cp_async16(dst + 2 * C::kCodes + lane * 16,
                               (lane < kScaleChunks ? k_from : v_from) + gap + (lane % kScaleChunks) * 16, take);
            }
        }
        cp_async_commit();
    };
    // The first keys are on their way while the queries are read.
#pragma unroll
    for (int n = 0; n < C::kStages - 1; ++n) {
        if constexpr (Q4) fetch4(n, n);
        else fetch16(n, n);
    }

    // Rows of this lane: n = g of each n tile as B operand, 2t and 2t + 1 as columns of the results.
    uint32_t qf[NT][KS][2];
    int pos[NT][2];
    float row_scale[NT][2];        // scale_log2, times what the row was divided by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int n = nt * 8 + g;
        const bool ok = n < rows;
        const int token = ok ? n / p.group : 0;
        const char* src = p.q + (it.q0 + token) * p.q_token_stride +
                          (it.head * p.group + (ok ? n - token * p.group : 0)) * p.q_head_stride;
        float factor = 1.f;
        if constexpr (Q4) {
            // d = (D/4) t + 4 ks + {0, 1} and {2, 3}
            uint2 raw[KS];
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) {
                const uint4 x = ok ? *(reinterpret_cast<const uint4*>(src + t * (D / 2)) + i) : make_uint4(0, 0, 0, 0);
                raw[2 * i] = make_uint2(x.x, x.y);
                raw[2 * i + 1] = make_uint2(x.z, x.w);
            }
            if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
                for (int i = 0; i < KS; ++i) qf[nt][i][0] = raw[i].x, qf[nt][i][1] = raw[i].y;
            } else {
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const float2 a = Pair<T>::unpack(raw[i].x), b = Pair<T>::unpack(raw[i].y);
                    amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
                }
                amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
                factor = row_divisor(amax);
                const float inv = 1.f / factor;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const float2 a = Pair<T>::unpack(raw[i].x), b = Pair<T>::unpack(raw[i].y);
                    qf[nt][i][0] = Pair<__half>::pack(a.x * inv, a.y * inv);
                    qf[nt][i][1] = Pair<__half>::pack(b.x * inv, b.y * inv);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t* s = reinterpret_cast<const uint32_t*>(src + 32 * i) + t;
                qf[nt][i][0] = ok ? s[0] : 0u;
                qf[nt][i][1] = ok ? s[4] : 0u;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int m = nt * 8 + 2 * t + c;
            pos[nt][c] = m < rows ? it.pos0 + m / p.group : -1;
            row_scale[nt][c] = p.scale_log2 * __shfl_sync(~0u, factor, (2 * t + c) * 4);
        }
    }

    float o[KS][NT][4];
    float mx[NT][2], sum[NT][2];      // what weights are taken relative to: maxima of scale_log2 * score, less kLift
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        mx[nt][0] = mx[nt][1] = -INFINITY;
        sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
        for (int m = 0; m < KS; ++m) o[m][nt][0] = o[m][nt][1] = o[m][nt][2] = o[m][nt][3] = 0.f;
    }

    const int key_of_row = Q4 ? (g >> 1) | ((g & 1) << 2) : g;     // the key in row g of S^T
    // NS slices: S^T, the softmax step and O^T, given the fragments of K and V.
    auto attend = [&](int first, auto&& k_frag, auto&& v_frag) {
        float s[NS][NT][4];
#pragma unroll
        for (int z = 0; z < NS; ++z) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[z][nt][0] = s[z][nt][1] = s[z][nt][2] = s[z][nt][3] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t a[4];
                k_frag(z, i, a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<M>(s[z][nt], a, qf[nt][i][0], qf[nt][i][1]);
            }
        }
        // Every key visible to every row: nothing to mask. (it.pos0 is the oldest row's position.)
        const int end = first + 16 * NS - 1;
        const bool whole = end <= it.pos0 && (last - first < p.window || end < p.sinks);
#pragma unroll
        for (int z = 0; z < NS; ++z)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[z][nt][e] *= row_scale[nt][e & 1];
        if (!whole) {
#pragma unroll
            for (int z = 0; z < NS; ++z)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!visible(p, pos[nt][e & 1], first + 16 * z + 8 * (e >> 1) + key_of_row)) s[z][nt][e] = -INFINITY;
        }
        float top[NT][2];
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                top[nt][c] = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
                for (int z = 1; z < NS; ++z) top[nt][c] = fmaxf(top[nt][c], fmaxf(s[z][nt][c], s[z][nt][c + 2]));
                top[nt][c] = fmaxf(top[nt][c], __shfl_xor_sync(~0u, top[nt][c], 4));
                top[nt][c] = fmaxf(top[nt][c], __shfl_xor_sync(~0u, top[nt][c], 8));
                top[nt][c] = fmaxf(top[nt][c], __shfl_xor_sync(~0u, top[nt][c], 16));
                grow |= top[nt][c] - mx[nt][c] > 8.f + kLift<M>;   // also from no key to a first one
            }
        // Rescale only when a row's maximum grows by more than 2^8: until then weights stay below that (2^15 with kLift).
        if (__any_sync(~0u, grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float next = fmaxf(mx[nt][c], top[nt][c] - kLift<M>);
                    const float shrink = exp2_approx(mx[nt][c] - (next == -INFINITY ? 0.f : next));
                    mx[nt][c] = next;
                    sum[nt][c] *= shrink;
#pragma unroll
                    for (int m = 0; m < KS; ++m) {
                        o[m][nt][c] *= shrink;
                        o[m][nt][c + 2] *= shrink;
                    }
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float base = mx[nt][c] == -INFINITY ? 0.f : mx[nt][c];
#pragma unroll
                for (int z = 0; z < NS; ++z) {
                    s[z][nt][c] = exp2_approx(s[z][nt][c] - base);
                    s[z][nt][c + 2] = exp2_approx(s[z][nt][c + 2] - base);
                    sum[nt][c] += s[z][nt][c] + s[z][nt][c + 2];
                }
            }
#pragma unroll
        for (int z = 0; z < NS; ++z) {
            uint32_t pw[NT][2];
            [[maybe_unused]] uint32_t pl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t w = Pair<M>::pack(s[z][nt][2 * h], s[z][nt][2 * h + 1]);
                    if constexpr (kTwoWeights) {
                        const float2 r = Pair<M>::unpack(w);
                        pl[nt][h] = transpose8x8(Pair<M>::pack(s[z][nt][2 * h] - r.x, s[z][nt][2 * h + 1] - r.y));
                    }
                    pw[nt][h] = transpose8x8(w);
                }
#pragma unroll
            for (int m = 0; m < KS; ++m) {
                uint32_t a[4];
                v_frag(z, m, a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816<M>(o[m][nt], a, pw[nt][0], pw[nt][1]);
                    if constexpr (kTwoWeights) mma16816<M>(o[m][nt], a, pl[nt][0], pl[nt][1]);
                }
            }
        }
    };

    int stage = 0;
    for (int n = 0; n < count; ++n) {
        cp_async_wait<C::kStages - 2>();
        __syncwarp();
        const int next = stage + C::kStages - 1;
        if constexpr (Q4) fetch4(n + C::kStages - 1, next >= C::kStages ? next - C::kStages : next);
        else fetch16(n + C::kStages - 1, next >= C::kStages ? next - C::kStages : next);
        const int first = first_of(kt.begin + n, 0);
        const uint32_t at = ring + stage * C::kStageBytes;
        if constexpr (!Q4) {
            const uint32_t v_at = at + 16 * D * 2;
            if (touched(first))
                attend(
                    first,
                    [&](int, int ks, uint32_t a[4]) {
                        const int r = lane & 15, c = 2 * ks + (lane >> 4);
                        ldmatrix4(a, at + r * (D * 2) + ((c ^ (r & 7)) << 4));
                    },
                    [&](int, int m, uint32_t a[4]) {
                        const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * m + ((lane >> 3) & 1);
                        ldmatrix4_t(a, v_at + r * (D * 2) + ((c ^ (r & 7)) << 4));
                    });
        } else {
            bool any = false;
#pragma unroll
            for (int z = 0; z < NS; ++z) any |= touched(first + 16 * z);
            if (any) {
                uint32_t kc[2][D / 32], sc[2][2], kd[2][4], vc[4][D / 64], vsc[2], vd[4][4];
                attend(
                    first,
                    [&](int z, int ks, uint32_t a[4]) {
                        // d = (D/4) t + 4 ks ... of the keys in rows g and g + 8; scale bytes: D = 128: 2t, 2t + 1
                        // (k steps 0-3, 4-7); D = 64: t.
                        if (ks == 0) {
                            const uint32_t from = at + z * 2 * (C::kCodes + C::kScales);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                ld_shared<D / 32>(kc[h], from + (g + 8 * h) * (D / 2) + t * (D / 8));
                                const uint32_t s = from + 2 * C::kCodes + (key_of_row + 8 * h) * (D / 16) + t * (D / 64);
                                const uint32_t both = D == 128 ? ld_shared_u16(s) : ld_shared_u8(s);
                                sc[h][0] = scales_to_half(__byte_perm(both, 0, 0x0000));
                                sc[h][1] = D == 128 ? scales_to_half(__byte_perm(both, 0, 0x1111)) : sc[h][0];
                            }
                        }
                        if ((ks & 1) == 0) {
                            codes_to_half(kc[0][ks / 2], kd[0]);
                            codes_to_half(kc[1][ks / 2], kd[1]);
                        }
                        const int b = 2 * (ks & 1), y = D == 128 ? ks / 4 : 0;
                        a[0] = mul_half2(kd[0][b], sc[0][y]);
                        a[1] = mul_half2(kd[1][b], sc[1][y]);
                        a[2] = mul_half2(kd[0][b + 1], sc[0][y]);
                        a[3] = mul_half2(kd[1][b + 1], sc[1][y]);
                    },
                    [&](int z, int m, uint32_t a[4]) {
                        // Byte m of a key's chunk holds d = (D/8) g + 2m (row g) and + 1 (row g + 8);
                        // pair the low and the high halves of two keys.
                        if (m == 0) {
                            const uint32_t from = at + z * 2 * (C::kCodes + C::kScales) + C::kCodes;
                            uint32_t b[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                const int key = t + 4 * u;
                                const int chunk = D == 128 ? (g >> 1) ^ (key & 2) : g >> 2;
                                ld_shared<D / 64>(vc[u], from + key * (D / 2) + chunk * 16 + (g * (D / 16)) % 16);
                                b[u] = ld_shared_u8(from + C::kCodes + C::kScales + key * (D / 16) + (D == 128 ? g : g / 2));
                            }
                            if (!filled(first + 16 * z))           // values that no row sees may be NaN: zeros
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    if (!wanted(first + 16 * z + t + 4 * u)) b[u] = 0;
                            vsc[0] = scales_to_half(b[0] | (b[1] << 8));
                            vsc[1] = scales_to_half(b[2] | (b[3] << 8));
                        }
                        if ((m & 3) == 0) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t w0 = vc[2 * h][m / 4], w1 = vc[2 * h + 1][m / 4];
                                codes_to_half((w0 & 0x0f0f0f0fu) | ((w1 << 4) & 0xf0f0f0f0u), vd[2 * h]);
                                codes_to_half(((w0 >> 4) & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u), vd[2 * h + 1]);
                            }
                        }
                        a[0] = mul_half2(vd[0][m & 3], vsc[0]);
                        a[1] = mul_half2(vd[1][m & 3], vsc[0]);
                        a[2] = mul_half2(vd[2][m & 3], vsc[1]);
                        a[3] = mul_half2(vd[3][m & 3], vsc[1]);
                    });
            }
        }
        __syncwarp();
        stage = stage + 1 == C::kStages ? 0 : stage + 1;
    }
    cp_async_wait<0>();

    // Join the four warps' results through shared memory.
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);                              // [warp][row][D]
    float* sm = so + kSplitWarps * kRows * D;                                // [warp][row][2]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float total = sum[nt][c];
            total += __shfl_xor_sync(~0u, total, 4);
            total += __shfl_xor_sync(~0u, total, 8);
            total += __shfl_xor_sync(~0u, total, 16);
            const int row = nt * 8 + 2 * t + c;
            if (g == 0) {
                sm[(warp * kRows + row) * 2] = mx[nt][c];
                sm[(warp * kRows + row) * 2 + 1] = total;
            }
            float* dst = so + (warp * kRows + row) * D;
#pragma unroll
            for (int m = 0; m < KS; ++m) {
                // 4-bit fragments hold d = (D/8) g + 2m + {0, 1}, the others 16m + g + {0, 8}.
                dst[Q4 ? (D / 8) * g + 2 * m : 16 * m + g] = o[m][nt][c];
                dst[Q4 ? (D / 8) * g + 2 * m + 1 : 16 * m + g + 8] = o[m][nt][c + 2];
            }
        }
    }
    __syncthreads();
    constexpr int kPairs = D / 2;
    bool spoiled = false;              // see mend_row
    for (int e = threadIdx.x; e < rows * kPairs; e += kSplitWarps * 32) {
        const int row = e / kPairs, d = 2 * (e - row * kPairs);
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, sm[(w * kRows + row) * 2]);
        const float base = top == -INFINITY ? 0.f : top;
        float total = 0.f, v[2] = {0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) {
            const float m = sm[(w * kRows + row) * 2];
            // A warp that saw no key of this row adds nothing, whatever its tiles held.
            const float f = exp2_approx(m - base);
            total = fmaf(f, sm[(w * kRows + row) * 2 + 1], total);
            const float2 x = *reinterpret_cast<const float2*>(so + (w * kRows + row) * D + d);
            v[0] = fmaf(f, x.x, v[0]);
            v[1] = fmaf(f, x.y, v[1]);
        }
        spoiled |= (isnan(v[0]) || isnan(v[1])) && !isnan(total);
        const int token = it.q0 + row / p.group, head = it.head * p.group + row % p.group;
        if (p.splits == 1) {
            const float inv = total > 0.f ? p.out_scale / total : (total == 0.f ? 0.f : total);
            const uint32_t packed = total == 0.f ? 0u : Pair<T>::pack(v[0] * inv, v[1] * inv);
            *reinterpret_cast<uint32_t*>(p.out + token * p.o_token_stride + head * p.o_head_stride + d * 2) = packed;
        } else {
            const int64_t at = (static_cast<int64_t>(token) * p.heads + head) * p.splits + it.split;
            *reinterpret_cast<float2*>(p.ws_o + at * D + d) = make_float2(v[0], v[1]);
            if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(top, total);
        }
    }
    if (__syncthreads_or(spoiled)) {
        int hint = -1;
        for (int row = warp; row < rows; row += kSplitWarps) {
            bool number = true;
            for (int w = 0; w < kSplitWarps; ++w) number &= !isnan(sm[(w * kRows + row) * 2 + 1]);
            if (number) mend_row<T, D, Q4>(p, it, kt, C::kKeys, row, false, &hint);
        }
    }
}

// Joins the splits' partial results: a CTA per row, its warps take every fourth split. The weights of
// the splits come first, so that the loads of the partial rows do not wait for each other.
constexpr int kJoinWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const __grid_constant__ AttnParams p) {
    __shared__ float weight[kMaxSplits];
    __shared__ float part[kJoinWarps][D];
    griddep_launch_dependents();
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x;
    const int token = static_cast<int>(row / p.heads), head = static_cast<int>(row - static_cast<int64_t>(token) * p.heads);
    if (p.cu != nullptr && (token < p.cu[0] || token >= p.cu[p.num_seqs])) return;     // no sequence's row
    const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + row * p.splits;
    // Every warp finds the maximum and the sum itself; warp 0 leaves the weights for all.
    constexpr int kPer = kMaxSplits / 32;
    float2 x[kPer];
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        x[k] = lane + 32 * k < p.splits ? ml[lane + 32 * k] : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, x[k].x);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        // A split that saw no key of the row counts nothing, whatever its values.
        const float f = x[k].y == 0.f ? 0.f : exp2_approx(x[k].x - base);
        total = fmaf(f, x[k].y, total);
        if (warp == 0) weight[lane + 32 * k] = f;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
    __syncthreads();
    constexpr int N = D / 32;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    const float* o = p.ws_o + row * p.splits * D + lane * N;
#pragma unroll 8
    for (int i = warp; i < p.splits; i += kJoinWarps) {
        const float f = weight[i];
        if (f == 0.f) continue;
        float v[N];
        if constexpr (N == 4) {
            const float4 w = __ldcg(reinterpret_cast<const float4*>(o + static_cast<int64_t>(i) * D));
            v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        } else {
            const float2 w = __ldcg(reinterpret_cast<const float2*>(o + static_cast<int64_t>(i) * D));
            v[0] = w.x, v[1] = w.y;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = fmaf(f, v[k], acc[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) part[warp][lane * N + k] = acc[k];
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const float inv = total == 0.f ? 0.f : p.out_scale / total;
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) a += part[w][2 * threadIdx.x], b += part[w][2 * threadIdx.x + 1];
        reinterpret_cast<uint32_t*>(p.out + token * p.o_token_stride + head * p.o_head_stride)[threadIdx.x] =
            total == 0.f ? 0u : Pair<T>::pack(a * inv, b * inv);
    }
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------

static cudaLaunchConfig_t launch_config(dim3 grid, int threads, int smem, cudaStream_t stream,
                                        cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

template <typename T, int D>
static int join(const AttnParams& p, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.heads;
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = launch_config(dim3(static_cast<unsigned>(rows)), kJoinWarps * 32, 0, stream, &attr);
    KVX_CUDA(cudaLaunchKernelEx(&cfg, attn_join_kernel<T, D>, p), "launch attention join kernel");
    return KVX_OK;
}

int launch_attn_join(const AttnParams& p, int head_dim, int dtype, cudaStream_t stream) {
    if (head_dim == 64) return dtype ? join<__half, 64>(p, stream) : join<__nv_bfloat16, 64>(p, stream);
    return dtype ? join<__half, 128>(p, stream) : join<__nv_bfloat16, 128>(p, stream);
}

template <typename T, int D, int NT, bool Q4>
static int run_split(const AttnParams& p, int device, cudaStream_t stream) {
    constexpr int smem = SplitConfig<D, NT, Q4>::kSmem;
    if constexpr (smem > 48 * 1024) {
        static std::atomic<uint64_t> done{0};               // devices that have the opt-in
        const uint64_t bit = 1ull << device;
        if (!(done.load(std::memory_order_relaxed) & bit)) {
            KVX_CUDA(cudaFuncSetAttribute(attn_split_kernel<T, D, NT, Q4>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          smem),
                     "set attention kernel shared memory");
            done.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = launch_config(dim3(p.tile_slots, p.kv_heads, p.splits), kSplitWarps * 32, smem, stream, &attr);
    KVX_CUDA(cudaLaunchKernelEx(&cfg, attn_split_kernel<T, D, NT, Q4>, p), "launch attention kernel");
    return KVX_OK;
}

template <typename T, int D, bool Q4>
static int run_rows(const AttnParams& p, int nt, int device, cudaStream_t stream) {
    switch (nt) {
        case 1: return run_split<T, D, 1, Q4>(p, device, stream);
        case 2: return run_split<T, D, 2, Q4>(p, device, stream);
        default: return run_split<T, D, 3, Q4>(p, device, stream);
    }
}

int launch_attn_split(const AttnParams& p, int head_dim, int dtype, bool q4, int nt, int device, cudaStream_t stream) {
    const auto run = head_dim == 64
                         ? (q4 ? (dtype ? run_rows<__half, 64, true> : run_rows<__nv_bfloat16, 64, true>)
                               : (dtype ? run_rows<__half, 64, false> : run_rows<__nv_bfloat16, 64, false>))
                         : (q4 ? (dtype ? run_rows<__half, 128, true> : run_rows<__nv_bfloat16, 128, true>)
                               : (dtype ? run_rows<__half, 128, false> : run_rows<__nv_bfloat16, 128, false>));
    return run(p, nt, device, stream);
}

}  // namespace kvx
