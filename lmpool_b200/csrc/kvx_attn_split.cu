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
// 4-bit cache: the fragments' order along head_dim is free as long as both
// operands agree, so a lane loads the codes it multiplies straight from global
// memory into registers (64 contiguous bytes per key, one slice ahead), turns
// them into fp16 and scales them there, exactly. Queries go to fp16 too, each row
// first divided by the power of two below its largest element.
// Weights: for a bf16 cache they are split in two bf16 numbers (2^-17 relative;
// the tensor cores have time to spare here), for fp16 and 4-bit rounded to fp16.

#include <atomic>
#include <climits>
#include <type_traits>

#include "kvx.h"
#include "kvx_attn.cuh"
#include "kvx_host.h"

namespace kvx {

constexpr int kSplitWarps = 4;
constexpr int kSplitKeys = 16 * kSplitWarps;   // keys of a tile

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
    const int n = take ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
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

template <int D, bool Q4>
struct SplitConfig {
    static constexpr int kStages = 3;
    static constexpr int kSliceBytes = 2 * 16 * D * 2;                       // K and V of 16 keys
    static constexpr int kRing = Q4 ? 0 : kStages * kSliceBytes * kSplitWarps;
    static constexpr int merge_bytes(int rows) { return kSplitWarps * rows * (D + 4) * 4; }
    static constexpr int smem(int rows) { return kRing > merge_bytes(rows) ? kRing : merge_bytes(rows); }
};

// A slice of the 4-bit cache as a lane holds it.
template <int D>
struct Q4Slice {
    uint32_t k[2][D / 32];     // keys g and g + 8: codes of d = (D/4) t ...
    uint32_t ks[2];            // their scales, one byte per 16 elements
    uint32_t v[4][D / 64];     // keys 2t, 2t+1, 2t+8, 2t+9: codes of d = (D/8) g ...
    uint32_t vs[2];            // scales of keys (2t, 2t+1) and (2t+8, 2t+9), two bytes each
};

template <typename T, int D, int NT, bool Q4>
__global__ void __launch_bounds__(kSplitWarps * 32) attn_split_kernel(const __grid_constant__ AttnParams p) {
    using M = typename std::conditional<Q4, __half, T>::type;     // type of the products' operands
    using C = SplitConfig<D, Q4>;
    constexpr int kRows = 8 * NT;
    constexpr int KS = D / 16;                                     // k steps of Q K^T, m tiles of V^T P^T
    constexpr bool kTwoWeights = !Q4 && std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(128) char smem[];
    griddep_launch_dependents();
    griddep_wait();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    AttnItem it = locate_item(p, blockIdx.x);
    it.head = blockIdx.y;
    it.split = blockIdx.z;
    if (it.tokens == 0) return;
    const KeyTiles kt = key_tiles<kSplitKeys>(p, it);
    const int rows = it.tokens * p.group;
    const int32_t* table = p.table + it.seq * p.table_stride;
    const int last = it.pos0 + it.tokens - 1;

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
    float mx[NT][2], sum[NT][2];      // maxima in units of scale_log2 * score
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        mx[nt][0] = mx[nt][1] = -INFINITY;
        sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
        for (int m = 0; m < KS; ++m) o[m][nt][0] = o[m][nt][1] = o[m][nt][2] = o[m][nt][3] = 0.f;
    }

    // One slice: S^T, the softmax step and O^T, given the fragments of K and V.
    auto attend = [&](int first, auto&& k_frag, auto&& v_frag) {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint32_t a[4];
            k_frag(i, a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<M>(s[nt], a, qf[nt][i][0], qf[nt][i][1]);
        }
        // Every key visible to every row: nothing to mask. (it.pos0 is the oldest row's position.)
        const bool whole = first + 15 <= it.pos0 && (last - first < p.window || first + 15 < p.sinks);
        uint32_t pw[NT][2];
        [[maybe_unused]] uint32_t pl[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x0 = s[nt][c] * row_scale[nt][c], x1 = s[nt][c + 2] * row_scale[nt][c];
                if (!whole) {
                    if (!visible(p, pos[nt][c], first + g)) x0 = -INFINITY;
                    if (!visible(p, pos[nt][c], first + g + 8)) x1 = -INFINITY;
                }
                float top = fmaxf(x0, x1);
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
                const float next = fmaxf(mx[nt][c], top);
                const float base = next == -INFINITY ? 0.f : next;
                const float shrink = exp2_approx(mx[nt][c] - base);
                mx[nt][c] = next;
                s[nt][c] = exp2_approx(x0 - base);
                s[nt][c + 2] = exp2_approx(x1 - base);
                sum[nt][c] = fmaf(sum[nt][c], shrink, s[nt][c] + s[nt][c + 2]);
#pragma unroll
                for (int m = 0; m < KS; ++m) {
                    o[m][nt][c] *= shrink;
                    o[m][nt][c + 2] *= shrink;
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t w = Pair<M>::pack(s[nt][2 * h], s[nt][2 * h + 1]);
                if constexpr (kTwoWeights) {
                    const float2 r = Pair<M>::unpack(w);
                    pl[nt][h] = transpose8x8(Pair<M>::pack(s[nt][2 * h] - r.x, s[nt][2 * h + 1] - r.y));
                }
                pw[nt][h] = transpose8x8(w);
            }
        }
#pragma unroll
        for (int m = 0; m < KS; ++m) {
            uint32_t a[4];
            v_frag(m, a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma16816<M>(o[m][nt], a, pw[nt][0], pw[nt][1]);
                if constexpr (kTwoWeights) mma16816<M>(o[m][nt], a, pl[nt][0], pl[nt][1]);
            }
        }
    };
    // Whether any row of the item sees key j: what no row sees is never read.
    auto wanted = [&](int j) {
        return j <= last && (it.pos0 - j < p.window || j < p.sinks);
    };
    // Whether a slice of 16 keys holds such a key.
    auto touched = [&](int first) {
        return first <= last && (it.pos0 - (first + 15) < p.window || first < p.sinks);
    };

    if constexpr (!Q4) {
        const uint32_t ring = smem_addr(smem) + warp * C::kStages * C::kSliceBytes;
        const int64_t head_off = it.head * p.head_stride;
        constexpr int kChunks = D / 8;                  // 16-byte chunks of a row
        constexpr int kRowsPerStep = 32 / kChunks;
        auto fetch = [&](int i, int stage) {
            if (i < kt.end) {
                const int first = kt.first_key<kSplitKeys>(i) + 16 * warp;
                int64_t off = -1;
                const int j = first + (lane & 15);
                if (wanted(j)) {
                    const int blk = block_of(p, j);
                    off = page_offset(p, table, blk);
                    if (off >= 0) off += (j - blk * p.block_size) * p.slot_stride + head_off;
                }
                const uint32_t dst = ring + stage * C::kSliceBytes;
                const int c = lane % kChunks;
#pragma unroll
                for (int r0 = 0; r0 < 16; r0 += kRowsPerStep) {
                    const int r = r0 + lane / kChunks;
                    const int64_t a = __shfl_sync(~0u, off, r);
                    const int64_t from = (a < 0 ? 0 : a) + c * 16;
                    const uint32_t to = dst + r * (D * 2) + ((c ^ (r & 7)) << 4);
                    cp_async16(to, p.k + from, a >= 0);
                    cp_async16(to + 16 * D * 2, p.v + from, a >= 0);
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < C::kStages - 1; ++i) fetch(kt.begin + i, i);
        int stage = 0;
        for (int i = kt.begin; i < kt.end; ++i) {
            cp_async_wait<C::kStages - 2>();
            __syncwarp();
            const int ahead = stage + C::kStages - 1;
            fetch(i + C::kStages - 1, ahead >= C::kStages ? ahead - C::kStages : ahead);
            const int first = kt.first_key<kSplitKeys>(i) + 16 * warp;
            const uint32_t k_at = ring + stage * C::kSliceBytes, v_at = k_at + 16 * D * 2;
            if (touched(first))
                attend(
                    first,
                    [&](int ks, uint32_t a[4]) {
                        const int r = lane & 15, c = 2 * ks + (lane >> 4);
                        ldmatrix4(a, k_at + r * (D * 2) + ((c ^ (r & 7)) << 4));
                    },
                    [&](int m, uint32_t a[4]) {
                        const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * m + ((lane >> 3) & 1);
                        ldmatrix4_t(a, v_at + r * (D * 2) + ((c ^ (r & 7)) << 4));
                    });
            __syncwarp();
            stage = stage + 1 == C::kStages ? 0 : stage + 1;
        }
        cp_async_wait<0>();
    } else {
        const int64_t head_off = it.head * p.head_stride;
        const int scales_at = p.block_size * (D / 2);
        auto fetch = [&](int i, Q4Slice<D>& x) {
            x.ks[0] = x.ks[1] = x.vs[0] = x.vs[1] = 0;
#pragma unroll
            for (int w = 0; w < D / 32; ++w) x.k[0][w] = x.k[1][w] = 0;
#pragma unroll
            for (int w = 0; w < D / 64; ++w) x.v[0][w] = x.v[1][w] = x.v[2][w] = x.v[3][w] = 0;
            if (i >= kt.end) return;
            const int first = kt.first_key<kSplitKeys>(i) + 16 * warp;
            if (!touched(first)) return;
            // block_size is a multiple of 16: a slice lies in one page.
            const int blk = block_of(p, first);
            const int64_t page = page_offset(p, table, blk);
            if (page < 0) return;
            const int off = first - blk * p.block_size;
            const char* kb = p.k + page + head_off;
            const char* vb = p.v + page + head_off;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = g + 8 * h;
                if (!wanted(first + key)) continue;
                const char* c = kb + (off + key) * (D / 2) + t * (D / 8);
                const char* s = kb + scales_at + (off + key) * (D / 16);
                if constexpr (D == 128) {
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(c));
                    x.k[h][0] = w.x, x.k[h][1] = w.y, x.k[h][2] = w.z, x.k[h][3] = w.w;
                    x.ks[h] = __ldg(reinterpret_cast<const uint16_t*>(s) + t);
                } else {
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(c));
                    x.k[h][0] = w.x, x.k[h][1] = w.y;
                    x.ks[h] = __ldg(reinterpret_cast<const uint8_t*>(s) + t);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int key = 2 * t + (u & 1) + 8 * (u >> 1);
                if (!wanted(first + key)) continue;
                const char* c = vb + (off + key) * (D / 2) + g * (D / 16);
                const char* s = vb + scales_at + (off + key) * (D / 16);
                if constexpr (D == 128) {
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(c));
                    x.v[u][0] = w.x, x.v[u][1] = w.y;
                    x.vs[u >> 1] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint8_t*>(s) + g)) << (8 * (u & 1));
                } else {
                    x.v[u][0] = __ldg(reinterpret_cast<const uint32_t*>(c));
                    x.vs[u >> 1] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint8_t*>(s) + g / 2)) << (8 * (u & 1));
                }
            }
        };
        Q4Slice<D> now, ahead;
        fetch(kt.begin, now);
        for (int i = kt.begin; i < kt.end; ++i) {
            fetch(i + 1, ahead);
            const int first = kt.first_key<kSplitKeys>(i) + 16 * warp;
            if (touched(first)) {
                // A lane's scales: D = 128: bytes 2t, 2t + 1 (k steps 0-3, 4-7); D = 64: byte t.
                uint32_t sc[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t lo = now.ks[h] & 0xff, hi = D == 128 ? now.ks[h] >> 8 : lo;
                    sc[h][0] = scales_to_half(lo | (lo << 8));
                    sc[h][1] = scales_to_half(hi | (hi << 8));
                }
                uint32_t kd[2][4];
                const uint32_t vsc[2] = {scales_to_half(now.vs[0]), scales_to_half(now.vs[1])};
                uint32_t vd[4][4];
                attend(
                    first,
                    [&](int ks, uint32_t a[4]) {
                        if ((ks & 1) == 0) {
                            codes_to_half(now.k[0][ks / 2], kd[0]);
                            codes_to_half(now.k[1][ks / 2], kd[1]);
                        }
                        const int b = 2 * (ks & 1), z = D == 128 ? ks / 4 : 0;
                        a[0] = mul_half2(kd[0][b], sc[0][z]);
                        a[1] = mul_half2(kd[1][b], sc[1][z]);
                        a[2] = mul_half2(kd[0][b + 1], sc[0][z]);
                        a[3] = mul_half2(kd[1][b + 1], sc[1][z]);
                    },
                    [&](int m, uint32_t a[4]) {
                        // Byte m of a key's chunk holds d = (D/8) g + 2m (row g) and + 1 (row g + 8);
                        // pair the low and the high halves of two neighbouring keys.
                        if ((m & 3) == 0) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t w0 = now.v[2 * h][m / 4], w1 = now.v[2 * h + 1][m / 4];
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
            now = ahead;
        }
    }

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
        if ((isnan(v[0]) || isnan(v[1])) && !isnan(total) && it.tokens > 1)
            visible_keys_only<T, D, Q4, 2>(p, it, kt, kSplitKeys, row, base, d, v);
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
}

// Joins the splits' partial results: one warp per row.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnParams p) {
    griddep_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (row >= static_cast<int64_t>(p.num_tokens) * p.heads) return;
    const int token = static_cast<int>(row / p.heads), head = static_cast<int>(row - static_cast<int64_t>(token) * p.heads);
    if (p.cu != nullptr && (token < p.cu[0] || token >= p.cu[p.num_seqs])) return;     // no sequence's row
    const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + row * p.splits;
    float top = -INFINITY;
    for (int i = lane; i < p.splits; i += 32) top = fmaxf(top, ml[i].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const float base = top == -INFINITY ? 0.f : top;
    constexpr int N = D / 32;
    float acc[N], total = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    for (int i = 0; i < p.splits; ++i) {
        const float2 x = ml[i];
        const float f = exp2_approx(x.x - base);
        total = fmaf(f, x.y, total);
        if (x.y == 0.f) continue;                       // this split saw no key of the row
        const float* o = p.ws_o + (row * p.splits + i) * D + lane * N;
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = fmaf(f, o[k], acc[k]);
    }
    const float inv = total == 0.f ? 0.f : p.out_scale / total;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + token * p.o_token_stride + head * p.o_head_stride) + lane * (N / 2);
#pragma unroll
    for (int k = 0; k < N; k += 2) dst[k / 2] = total == 0.f ? 0u : Pair<T>::pack(acc[k] * inv, acc[k + 1] * inv);
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
    cudaLaunchConfig_t cfg = launch_config(dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, stream, &attr);
    KVX_CUDA(cudaLaunchKernelEx(&cfg, attn_join_kernel<T, D>, p), "launch attention join kernel");
    return KVX_OK;
}

int launch_attn_join(const AttnParams& p, int head_dim, int dtype, cudaStream_t stream) {
    if (head_dim == 64) return dtype ? join<__half, 64>(p, stream) : join<__nv_bfloat16, 64>(p, stream);
    return dtype ? join<__half, 128>(p, stream) : join<__nv_bfloat16, 128>(p, stream);
}

template <typename T, int D, int NT, bool Q4>
static int run_split(const AttnParams& p, int device, cudaStream_t stream) {
    constexpr int smem = SplitConfig<D, Q4>::smem(8 * NT);
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
        default: return run_split<T, D, 4, Q4>(p, device, stream);
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
