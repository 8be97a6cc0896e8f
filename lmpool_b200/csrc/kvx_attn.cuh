// Shared by the paged-attention kernels: launch parameters, the cut of a call
// into work items, the keys an item reads, tensor-core and 4-bit helpers.
//
// Row r of an item is query head (r % G) of its kv head's group and token
// (r / G) of its run of tokens, so that all rows of an item share one kv head
// and every key is read once for G heads. Token t of sequence s stands at
// position p = context_len - q_len + t and sees key j when
//     j <= p  and  (p - j < window  or  j < sinks).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "kvx.h"
#include "kvx_device.cuh"

namespace kvx {

constexpr int kMaxSplits = 64;

struct AttnParams {
    const char* q;
    char* out;
    const char* k;
    const char* v;
    int64_t q_token_stride, q_head_stride;    // bytes
    int64_t o_token_stride, o_head_stride;
    int64_t block_stride, slot_stride, head_stride;
    int64_t num_blocks;
    const int32_t* table;
    int64_t table_stride;                     // entries
    const int32_t* ctx;
    const int32_t* cu;                        // nullptr: one token per sequence
    int32_t* status;
    float* ws_o;                              // [tokens * heads][splits][D], not yet divided by the sum
    float* ws_ml;                             // [tokens * heads][splits][2]: what weights are relative to (scale_log2 * score), sum
    float scale_log2;                         // scale * log2(e) (* k_scale of a 4-bit cache)
    float out_scale;                          // v_scale of a 4-bit cache, else 1
    int32_t table_width, block_size, block_shift;   // block_shift < 0: not a power of two
    int32_t num_seqs, num_tokens;
    int32_t heads, kv_heads, group;
    int32_t window, sinks;                    // window: INT_MAX when there is none
    int32_t splits, min_tiles;                // key tiles of a split, at least
    int32_t tile_tokens;                      // tokens of an item
    int32_t tile_slots;                       // item slots per (kv head, split)
    int32_t out_wide;                         // output rows start at multiples of 32 bytes
};

struct AttnItem {
    int seq;
    int q0;        // first token row
    int tokens;    // tokens of this item (0: nothing to do)
    int pos0;      // position of the first token (negative: before the context)
    int head;      // kv head
    int split;
};

// Length of sequence s's context, held in what its table can address.
__device__ __forceinline__ int context_of(const AttnParams& p, int s) {
    const int64_t cap = static_cast<int64_t>(p.table_width) * p.block_size;
    int64_t c = p.ctx[s];
    if (c < 0 || c > cap) {
        atomicOr(p.status, KVX_DEV_BAD_LEN);
        c = c < 0 ? 0 : cap;
    }
    return static_cast<int>(c);
}

// Flags cu_seqlens_q entries of sequence s that are out of order or range. The search below may pass over one.
__device__ __forceinline__ void check_offsets(const AttnParams& p, int s) {
    const int a = p.cu[s], b = p.cu[s + 1];
    if (a < 0 || b < a || b > p.num_tokens) atomicOr(p.status, KVX_DEV_BAD_LEN);
}

// Tile slot `x` of a call. Without cu_seqlens a slot is a sequence. With them
// the slots of sequence s start at cu[s] / tile + s: that leaves every
// sequence at least ceil(len / tile) of them, needs no prefix sum and no
// host copy of the lengths; spare slots hold no tokens.
__device__ __forceinline__ AttnItem locate_item(const AttnParams& p, int x) {
    AttnItem it;
    it.tokens = 0;
    it.head = 0;
    it.split = 0;
    if (p.cu == nullptr) {
        it.seq = x;
        it.q0 = x;
        it.tokens = 1;
        it.pos0 = context_of(p, x) - 1;
        return it;
    }
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu[mid] / p.tile_tokens + mid <= x) lo = mid;
        else hi = mid - 1;
    }
    it.seq = lo;
    const int a = p.cu[lo], b = p.cu[lo + 1];
    if (a < 0 || b < a || b > p.num_tokens) {
        atomicOr(p.status, KVX_DEV_BAD_LEN);
        it.q0 = it.pos0 = 0;
        return it;
    }
    const int64_t first = static_cast<int64_t>(x - (a / p.tile_tokens + lo)) * p.tile_tokens;
    it.q0 = static_cast<int>(a + (first < 0 ? 0 : first));
    it.pos0 = 0;
    if (first < 0 || first >= b - a) return it;
    it.tokens = static_cast<int>(b - a - first < p.tile_tokens ? b - a - first : p.tile_tokens);
    it.pos0 = static_cast<int>(context_of(p, lo) - (b - a) + first);
    return it;
}

// Keys of an item in tiles of KT: the tiles that hold a sink, then those from
// the oldest key of the first token's window to the last token's own key.
struct KeyTiles {
    int head;      // leading tiles (sinks)
    int skip;      // tiles between them and the window
    int begin, end;   // this split's range of tile numbers
    template <int KT>
    __device__ __forceinline__ int first_key(int i) const {
        return (i < head ? i : i + skip) * KT;
    }
};

template <int KT>
__device__ __forceinline__ KeyTiles key_tiles(const AttnParams& p, const AttnItem& it) {
    KeyTiles t;
    const int last = it.pos0 + it.tokens - 1;      // newest visible key
    t.head = t.skip = t.begin = t.end = 0;
    if (it.tokens == 0 || last < 0) return t;
    const int total = last / KT + 1;
    // A first token that stands before the context sees nothing: the window that counts is the one
    // of the first token with a position.
    const int first = it.pos0 < 0 ? 0 : it.pos0;
    const int lo = first >= p.window ? first - p.window + 1 : 0;
    const int low_tile = lo / KT;
    const int sink_tiles = p.sinks > 0 ? (min(p.sinks, last + 1) - 1) / KT + 1 : 0;
    t.head = min(sink_tiles, low_tile);
    t.skip = low_tile - t.head;
    const int n = total - t.skip;
    // A split of its own only for enough keys: the host knows no lengths, only what a table can hold.
    const int per = max((n + p.splits - 1) / p.splits, p.min_tiles);
    t.begin = min(n, it.split * per);
    t.end = min(n, t.begin + per);
    return t;
}

// Whether key j is visible to a token at position pos.
__device__ __forceinline__ bool visible(const AttnParams& p, int pos, int j) {
    return j <= pos && (pos - j < p.window || j < p.sinks);
}

// Byte offset of page `blk` of a sequence in the cache, or -1 (flagged).
__device__ __forceinline__ int64_t page_offset(const AttnParams& p, const int32_t* table, int blk) {
    const int64_t id = blk < p.table_width ? table[blk] : -1;
    if (id < 0 || id >= p.num_blocks) {
        atomicOr(p.status, KVX_DEV_BAD_SRC_ID);
        return -1;
    }
    return id * p.block_stride;
}

__device__ __forceinline__ int block_of(const AttnParams& p, int j) {
    return p.block_shift >= 0 ? j >> p.block_shift : j / p.block_size;
}

// 16 bytes into shared memory, zeros unless `take`.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
    const int n = take ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// ---------------------------------------------------------------------------
// Numbers
// ---------------------------------------------------------------------------

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
    static constexpr int kInf = 0x7f80;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t x) {
        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    }
};
template <>
struct Pair<__half> {
    static constexpr int kInf = 0x7c00;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t x) {
        __half2 h;
        memcpy(&h, &x, 4);
        return __half22float2(h);
    }
};

// Four codes pairs (8 codes, low half of a byte first) as f16x2; the levels
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives are exact in fp16.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t out[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3])
        : "r"(w));
}
// Two e4m3 scales (exact in fp16).
__device__ __forceinline__ uint32_t scales_to_half(uint32_t two) {
    uint32_t r;
    const uint16_t v = static_cast<uint16_t>(two);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// code * scale has at most six significant bits and lies in [2^-10, 2688]: exact.
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Weights are 2^(score - maximum + this), a factor that the division by their sum takes out again. As fp16 (a 4-bit cache's
// products and fp16 ones) a weight is off by 2^-25 at least, however small it is: 131070 keys of 2^-26 of the largest weight,
// 0.2 % of a row behind a strong sink, were all rounded to 0. Seven binades higher the largest still fits (a maximum may be
// stale by 2^8: 2^15) and the same weights are exact. bf16 reaches as far down as fp32.
template <typename M>
constexpr float kLift = std::is_same<M, __half>::value ? 7.f : 0.f;

// What a row of bf16 queries is divided by on its way to fp16: the power of two below
// its largest element, which keeps every element within 2^-25 of that one; 1 for
// rows that are zero, below 2^-100 or not finite.
__device__ __forceinline__ float row_divisor(float amax) {
    const uint32_t e = __float_as_uint(amax) & 0x7f800000u;
    return e < 0x0d800000u || e == 0x7f800000u ? 1.f : __uint_as_float(e);
}

// ---------------------------------------------------------------------------
// Rows that a masked value spoiled
// ---------------------------------------------------------------------------
//
// A product with a masked key is skipped in the formula, but a tile multiplies every row with every key: weight 0 times
// a value that is infinite or NaN gives NaN in rows that do not see that key. So does, for an infinity that a row sees, a
// weight that rounds to 0 or the second part of a weight in two. Such elements (NaN although the row's sum
// is a number) are computed again from the row's visible keys alone, by a warp a row, when no other warp waits for it. An
// element that sees values that are not finite has its result from those alone, and a row all of whose elements are NaN by
// them is left there. Only inputs that are not finite come here.

// A lane's elements of a row of the cache, lane * D / 32 and following, as fp32; zeros for a bad page.
template <typename T, int D, bool Q4>
__device__ __forceinline__ void lane_elements(const AttnParams& p, const char* plane, int64_t page, int off, int head,
                                              float (&v)[D / 32]) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const char* base = plane + page + head * p.head_stride;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        float2 x = make_float2(0.f, 0.f);
        if (page >= 0) {
            if constexpr (Q4) {
                const uint8_t* b = reinterpret_cast<const uint8_t*>(base);
                // The byte four times over: of a word whose upper bytes are known to be 0, nvcc 12.9 makes zeros.
                uint32_t h[4];
                codes_to_half(b[off * (D / 2) + lane * (N / 2) + i] * 0x01010101u, h);
                const uint32_t scale = b[p.block_size * (D / 2) + off * (D / 16) + lane * N / 16];
                x = Pair<__half>::unpack(mul_half2(h[0], scales_to_half(scale | (scale << 8))));
            } else {
                x = Pair<T>::unpack(reinterpret_cast<const uint32_t*>(base + off * p.slot_stride)[lane * (N / 2) + i]);
            }
        }
        v[2 * i] = x.x;
        v[2 * i + 1] = x.y;
    }
}

// The product of a query row with a row of the cache, by one lane; 0 for a bad page.
template <typename T, int D, bool Q4>
__device__ __forceinline__ float row_product(const AttnParams& p, const T* q, int64_t page, int off, int head) {
    if (page < 0) return 0.f;
    const char* base = p.k + page + head * p.head_stride;
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {                               // 8 elements at a time
        const uint4 x = reinterpret_cast<const uint4*>(q)[c];
        const uint32_t a[4] = {x.x, x.y, x.z, x.w};
        uint32_t k[4];
        if constexpr (Q4) {
            codes_to_half(reinterpret_cast<const uint32_t*>(base + off * (D / 2))[c], k);
            const uint32_t scale = reinterpret_cast<const uint8_t*>(base)[p.block_size * (D / 2) + off * (D / 16) + c / 2];
#pragma unroll
            for (int i = 0; i < 4; ++i) k[i] = mul_half2(k[i], scales_to_half(scale | (scale << 8)));
        } else {
            const uint4 y = reinterpret_cast<const uint4*>(base + off * p.slot_stride)[c];
            k[0] = y.x, k[1] = y.y, k[2] = y.z, k[3] = y.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 u = Pair<T>::unpack(a[i]), v = Pair<typename std::conditional<Q4, __half, T>::type>::unpack(k[i]);
            s = fmaf(u.x, v.x, s);
            s = fmaf(u.y, v.y, s);
        }
    }
    return s;
}

// In a 16-bit output, a NaN that is to be computed again (conversions give 0x7fff).
template <typename T>
__device__ __forceinline__ constexpr uint16_t marked_nan() {
    return std::is_same<T, __half>::value ? 0x7e01 : 0x7fc1;
}

// A warp's work on one finished row: its NaN elements (the marked ones of an output row with `marked`) again. `hint` is a
// key whose values gave NaN in the row before: the next row mostly has its NaN from there too.
template <typename T, int D, bool Q4>
__device__ __noinline__ void mend_row(const AttnParams& p, const AttnItem& it, const KeyTiles& kt, int tile_keys, int row,
                                      bool marked, int* hint) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const int token = row / p.group, head = it.head * p.group + row - token * p.group;
    const int pos = it.pos0 + token;
    uint16_t* out = reinterpret_cast<uint16_t*>(p.out + (it.q0 + token) * p.o_token_stride + head * p.o_head_stride) + lane * N;
    const int64_t at = (static_cast<int64_t>(it.q0 + token) * p.heads + head) * p.splits + it.split;
    float* part = p.ws_o + at * D + lane * N;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool nan = p.splits > 1 ? isnan(part[i]) : marked ? out[i] == marked_nan<T>() : (out[i] & 0x7fff) > Pair<T>::kInf;
        bad |= static_cast<uint32_t>(nan) << i;
    }
    if (!__any_sync(~0u, bad)) return;

    // What the element has of values that are not finite: their sum decides it, whatever the weights.
    float odd[N], acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) odd[i] = acc[i] = 0.f;
    auto covered = [&]() {
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) nan |= static_cast<uint32_t>(isnan(odd[i])) << i;
        return __all_sync(~0u, (bad & ~nan) == 0);
    };
    const int32_t* table = p.table + it.seq * p.table_stride;
    bool done = false;
    if (*hint >= 0 && visible(p, pos, *hint)) {
        const int blk = block_of(p, *hint);
        float v[N];
        lane_elements<T, D, Q4>(p, p.v, page_offset(p, table, blk), *hint - blk * p.block_size, it.head, v);
#pragma unroll
        for (int i = 0; i < N; ++i) odd[i] = isnan(v[i]) ? v[i] : 0.f;
        done = covered();
        if (!done)
#pragma unroll
            for (int i = 0; i < N; ++i) odd[i] = 0.f;
    }
    // 32 keys at a time: a lane finds the page and the score of one of them, then their values come row by row.
    const T* q = reinterpret_cast<const T*>(p.q + (it.q0 + token) * p.q_token_stride + head * p.q_head_stride);
    float m = -INFINITY, sum = 0.f;                                 // this lane's part of the sum
    for (int n = kt.begin * (tile_keys / 32); n < kt.end * (tile_keys / 32) && !done; ++n) {
        const int tile = n / (tile_keys / 32);
        const int first = (tile < kt.head ? tile : tile + kt.skip) * tile_keys + 32 * (n - tile * (tile_keys / 32));
        const int j = first + lane;
        const bool see = visible(p, pos, j);
        const uint32_t seen = __ballot_sync(~0u, see);
        if (!seen) continue;
        const int blk = block_of(p, j), off = j - blk * p.block_size;
        const int64_t page = see ? page_offset(p, table, blk) : -1;
        const float s = see ? row_product<T, D, Q4>(p, q, page, off, it.head) * p.scale_log2 : -INFINITY;
        float next = s;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) next = fmaxf(next, __shfl_xor_sync(~0u, next, d));
        next = fmaxf(next, m);
        const float base = next == -INFINITY ? 0.f : next, shrink = exp2f(m - base), w = exp2f(s - base);
        m = next;
        sum = fmaf(sum, shrink, w);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] *= shrink;
        uint32_t nan = 0;                                           // keys with a NaN among this lane's elements
#pragma unroll 8
        for (int u = 0; u < 32; ++u) {
            float v[N];
            lane_elements<T, D, Q4>(p, p.v, __shfl_sync(~0u, page, u), __shfl_sync(~0u, off, u), it.head, v);
            const float weight = __shfl_sync(~0u, w, u);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool fine = fabsf(v[i]) < INFINITY;
                acc[i] = fmaf(weight, fine ? v[i] : 0.f, acc[i]);
                odd[i] += fine ? 0.f : v[i];
                nan |= static_cast<uint32_t>(isnan(v[i])) << u;
            }
        }
        done = covered();
        nan = __reduce_or_sync(~0u, nan);
        if (done && nan) *hint = first + __ffs(nan) - 1;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    // A partial result is relative to what the split's other elements are.
    const float mine = m == -INFINITY ? 0.f : m;
    float factor = sum > 0.f ? p.out_scale / sum : 0.f;
    if (p.splits > 1) {
        const float ref = p.ws_ml[at * 2];
        factor = exp2f(mine - (ref == -INFINITY ? 0.f : ref));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float x = odd[i] == 0.f ? acc[i] * factor : odd[i];
        if (!(bad & (1u << i))) continue;
        if (p.splits > 1) part[i] = x;
        else reinterpret_cast<T*>(out)[i] = static_cast<T>(x);
    }
}

// ---------------------------------------------------------------------------
// Launches (one translation unit per kernel family)
// ---------------------------------------------------------------------------

// Rows are few: keys split over CTAs and warps (kvx_attn_split.cu). An item has 8 * nt rows (nt = 1 to 3).
int launch_attn_split(const AttnParams& p, int head_dim, int dtype, bool q4, int nt, int device, cudaStream_t stream);
// Rows are many: 256-row tiles on the tensor cores (kvx_attn_tile.cu).
int launch_attn_tile(const AttnParams& p, int head_dim, int dtype, bool q4, int device, int sms, cudaStream_t stream);
// Joins the splits of either (kvx_attn_split.cu).
int launch_attn_join(const AttnParams& p, int head_dim, int dtype, cudaStream_t stream);

}  // namespace kvx
