// Rows into and out of the 4-bit paged cache (format: include/kvx.h).
//
// Both kernels give a thread one group of 16 elements: 32 bytes on the 16-bit
// side, 8 bytes of codes and one scale byte on the 4-bit side. Floor: HBM
// bytes, 2 + 9/16 per element; at a decode step's 256 tokens a launch's latency.
// Measured, 8 kv heads of 128, rows stored and loaded again, two calls: 16384 tokens 42 us, 4.1 TB/s, 0.62 of the
// copy rate (issue slots 80 % busy in the store, 68 % in the load: the conversion's instructions come first, then the
// pieces: a row of a head is 64 bytes of codes and 8 of scales in a page); 256 tokens 23 us, the host's two calls.
//
// The codes are those of exact arithmetic. amax / 6 is divided in IEEE fp32: an
// exact tie between two e4m3 values divides exactly, and a 16-bit amax that is no
// tie stays 2^-13 (relative) away from it. x / s is x * (1 / s), off by at most
// two fp32 steps, then rounded to 19 significant bits: where x is exactly a
// border t * s (t = 0.25, 0.75, ... 5) that gives t back and the tie goes to the
// even code; where it is not, t * s has at most 7 and x at most 11 significant
// bits, so x / s is at least 2^-12 (relative) away from t and stays on its side.

#include <climits>

#include "kvx.h"
#include "kvx_attn.cuh"
#include "kvx_host.h"

namespace kvx {

constexpr int kQ4Threads = 256;

struct Q4Params {
    const char* key;
    const char* value;
    char* key_out;
    char* value_out;
    char* k_cache;
    char* v_cache;
    int64_t key_token_stride, value_token_stride;   // bytes
    int64_t block_stride;
    const int64_t* slots;
    int64_t num_slots;
    int32_t rows;                                   // 2 * tokens: K and V of a token follow each other
    int32_t block_rows;                             // rows of a CTA
    int32_t block_size, block_shift, heads, head_dim;   // block_shift < 0: not a power of two
    int32_t row_groups;                             // heads * head_dim / 16
    float k_mul, v_mul;                             // store: 1 / scale, load: scale
    int32_t* status;
};

struct Q4Place {
    int64_t codes, scale;    // byte offsets of the group in its plane
};

// This thread's plane, token and group of the row; false where there is none.
__device__ __forceinline__ bool q4_item(const Q4Params& p, int* plane, int64_t* token, int* group) {
    const int in_block = static_cast<int>(threadIdx.x) / p.row_groups;
    const int row = static_cast<int>(blockIdx.x) * p.block_rows + in_block;
    *group = static_cast<int>(threadIdx.x) - in_block * p.row_groups + static_cast<int>(blockIdx.y) * kQ4Threads;
    *plane = row & 1;
    *token = row >> 1;
    return in_block < p.block_rows && row < p.rows && *group < p.row_groups;
}

__device__ __forceinline__ Q4Place q4_place(const Q4Params& p, int64_t slot, int group) {
    const int per_head = p.head_dim / 16;
    const int head = group / per_head, g = group - head * per_head;
    int64_t blk;
    if (p.block_shift >= 0) blk = slot >> p.block_shift;
    else if (p.num_slots <= INT_MAX) blk = static_cast<int>(slot) / p.block_size;
    else blk = slot / p.block_size;
    const int off = static_cast<int>(slot - blk * p.block_size);
    const int64_t run = blk * p.block_stride + static_cast<int64_t>(head) * p.block_size * (p.head_dim / 16 * 9);
    Q4Place a;
    a.codes = run + off * (p.head_dim / 2) + g * 8;
    a.scale = run + static_cast<int64_t>(p.block_size) * (p.head_dim / 2) + off * per_head + g;
    return a;
}

__device__ __forceinline__ bool q4_slot(const Q4Params& p, int64_t slot, int group, int plane) {
    if (slot == -1) return false;
    if (slot < -1 || slot >= p.num_slots) {
        if (group == 0 && plane == 0) atomicOr(p.status, KVX_DEV_BAD_SLOT);
        return false;
    }
    return true;
}

template <typename T>
__global__ void __launch_bounds__(kQ4Threads) store_q4_kernel(const __grid_constant__ Q4Params p) {
    griddep_launch_dependents();
    griddep_wait();
    int plane, group;
    int64_t token;
    if (!q4_item(p, &plane, &token, &group)) return;
    const int64_t slot = ld_cg(p.slots + token);
    const char* src = plane ? p.value + token * p.value_token_stride : p.key + token * p.key_token_stride;
    uint32_t raw[8];
    const uint4 lo = ld_cg(reinterpret_cast<const uint4*>(src + group * 32));
    const uint4 hi = ld_cg(reinterpret_cast<const uint4*>(src + group * 32) + 1);
    if (!q4_slot(p, slot, group, plane)) return;
    raw[0] = lo.x, raw[1] = lo.y, raw[2] = lo.z, raw[3] = lo.w;
    raw[4] = hi.x, raw[5] = hi.y, raw[6] = hi.z, raw[7] = hi.w;
    const float mul = plane ? p.v_mul : p.k_mul;
    // The largest magnitude: the bits of bf16 and of fp16 without their sign are ordered as numbers, NaN above infinity.
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_u16x2(most, raw[i] & 0x7fff7fffu);
    most = max(most & 0xffffu, most >> 16);
    const bool finite = most < Pair<T>::kInf;
    const float amax = Pair<T>::unpack(most).x * mul;               // may overflow: the scale saturates
    uint16_t scale2;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(scale2) : "f"(__fdiv_rn(amax, 6.f)));
    const float s = Pair<__half>::unpack(scales_to_half(scale2)).x;
    const float r = s > 0.f ? __frcp_rn(s) * mul : 0.f;         // mul is a power of two: as exact as 1 / s
    uint32_t codes[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 v = Pair<T>::unpack(raw[4 * i + k]);
            y[2 * k] = __uint_as_float((__float_as_uint(v.x * r) + 0x10u) & ~0x1fu);
            y[2 * k + 1] = __uint_as_float((__float_as_uint(v.y * r) + 0x10u) & ~0x1fu);
        }
        asm("{\n\t.reg .b8 a, b, c, d;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
            "mov.b32 %0, {a, b, c, d};\n\t}"
            : "=r"(codes[i])
            : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    }
    if (!finite) scale2 = 0x7f;
    if (!finite || s == 0.f) codes[0] = codes[1] = 0;
    char* cache = plane ? p.v_cache : p.k_cache;
    const Q4Place a = q4_place(p, slot, group);
    *reinterpret_cast<uint2*>(cache + a.codes) = make_uint2(codes[0], codes[1]);
    *reinterpret_cast<uint8_t*>(cache + a.scale) = static_cast<uint8_t>(scale2);
}

template <typename T>
__global__ void __launch_bounds__(kQ4Threads) load_q4_kernel(const __grid_constant__ Q4Params p) {
    griddep_launch_dependents();
    griddep_wait();
    int plane, group;
    int64_t token;
    if (!q4_item(p, &plane, &token, &group)) return;
    const int64_t slot = ld_cg(p.slots + token);
    uint32_t out[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (q4_slot(p, slot, group, plane)) {
        const char* cache = plane ? p.v_cache : p.k_cache;
        const float mul = plane ? p.v_mul : p.k_mul;
        const Q4Place a = q4_place(p, slot, group);
        const uint2 codes = ld_cg(reinterpret_cast<const uint2*>(cache + a.codes));
        const uint32_t scale = ld_cg(reinterpret_cast<const uint8_t*>(cache + a.scale));
        const uint32_t s2 = scales_to_half(scale | (scale << 8));
        uint32_t h[8];
        codes_to_half(codes.x, h);
        codes_to_half(codes.y, h + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = Pair<__half>::unpack(mul_half2(h[i], s2));
            out[i] = Pair<T>::pack(v.x * mul, v.y * mul);
        }
    }
    char* dst = plane ? p.value_out + token * p.value_token_stride : p.key_out + token * p.key_token_stride;
    uint4* d = reinterpret_cast<uint4*>(dst + group * 32);
    d[0] = make_uint4(out[0], out[1], out[2], out[3]);
    d[1] = make_uint4(out[4], out[5], out[6], out[7]);
}

static int q4_launch(bool store, int32_t device, int32_t dtype, const void* key, const void* value,
                     int64_t key_token_stride, int64_t value_token_stride, const void* k_cache, const void* v_cache,
                     int64_t block_stride, const int64_t* slots, int64_t num_tokens, int64_t num_blocks,
                     int32_t block_size, int32_t kv_heads, int32_t head_dim, float k_scale, float v_scale,
                     int32_t* status, void* stream) {
    if (dtype != 0 && dtype != 1) return fail(KVX_EINVAL, "dtype must be 0 (bf16) or 1 (fp16)");
    if (num_tokens < 0) return fail(KVX_EINVAL, "negative token count");
    if (num_blocks <= 0) return fail(KVX_EINVAL, "num_blocks must be > 0");
    if (block_size <= 0 || block_size % 16 != 0) return fail(KVX_EINVAL, "block_size must be a multiple of 16");
    if (head_dim <= 0 || head_dim % 16 != 0 || head_dim > 256)
        return fail(KVX_EINVAL, "head_dim must be a multiple of 16, at most 256");
    if (kv_heads <= 0 || kv_heads > 65536) return fail(KVX_EINVAL, "kv_heads must be in [1, 65536]");
    if (static_cast<int64_t>(block_size) * head_dim > INT_MAX / 2)
        return fail(KVX_EINVAL, "block_size * head_dim is too large");
    if (!power_of_two(k_scale) || !power_of_two(v_scale))
        return fail(KVX_EINVAL, "k_scale and v_scale must be powers of two in [2^-64, 2^63]");
    if (status == nullptr) return fail(KVX_EINVAL, "status_dev is NULL");
    if (num_tokens == 0) return KVX_OK;
    if (!key || !value || !k_cache || !v_cache || !slots) return fail(KVX_EINVAL, "NULL tensor pointer");
    const uint64_t bits = reinterpret_cast<uint64_t>(key) | reinterpret_cast<uint64_t>(value) |
                          reinterpret_cast<uint64_t>(k_cache) | reinterpret_cast<uint64_t>(v_cache) |
                          static_cast<uint64_t>(key_token_stride) | static_cast<uint64_t>(value_token_stride) |
                          static_cast<uint64_t>(block_stride);
    if (bits & 15) return fail(KVX_EINVAL, "addresses and strides must be multiples of 16 bytes");
    Q4Params p;
    p.key = static_cast<const char*>(key);
    p.value = static_cast<const char*>(value);
    p.key_out = const_cast<char*>(p.key);
    p.value_out = const_cast<char*>(p.value);
    p.k_cache = const_cast<char*>(static_cast<const char*>(k_cache));
    p.v_cache = const_cast<char*>(static_cast<const char*>(v_cache));
    p.key_token_stride = key_token_stride;
    p.value_token_stride = value_token_stride;
    p.block_stride = block_stride;
    p.slots = slots;
    p.num_slots = num_blocks * block_size;
    p.block_size = block_size;
    p.block_shift = -1;
    if ((block_size & (block_size - 1)) == 0)
        for (p.block_shift = 0; (1 << p.block_shift) < block_size;) ++p.block_shift;
    p.heads = kv_heads;
    p.head_dim = head_dim;
    p.row_groups = kv_heads * (head_dim / 16);
    if (num_tokens > INT_MAX / 4) return fail(KVX_EINVAL, "too many tokens");
    p.rows = static_cast<int32_t>(2 * num_tokens);
    p.block_rows = p.row_groups < kQ4Threads ? kQ4Threads / p.row_groups : 1;
    p.k_mul = store ? 1.f / k_scale : k_scale;
    p.v_mul = store ? 1.f / v_scale : v_scale;
    p.status = status;
    const dim3 grid(static_cast<unsigned>((p.rows + p.block_rows - 1) / p.block_rows),
                    static_cast<unsigned>((p.row_groups + kQ4Threads - 1) / kQ4Threads));
    if (grid.y > 65535) return fail(KVX_EINVAL, "rows of kv_heads * head_dim are too long");
    KVX_DEVICE_GUARD(device);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kQ4Threads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e;
    if (store)
        e = dtype ? cudaLaunchKernelEx(&cfg, store_q4_kernel<__half>, p)
                  : cudaLaunchKernelEx(&cfg, store_q4_kernel<__nv_bfloat16>, p);
    else
        e = dtype ? cudaLaunchKernelEx(&cfg, load_q4_kernel<__half>, p)
                  : cudaLaunchKernelEx(&cfg, load_q4_kernel<__nv_bfloat16>, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return cuda_fail(e, store ? "launch store_kvcache_q4 kernel" : "launch load_kvcache_q4 kernel");
    }
    return KVX_OK;
}

}  // namespace kvx

using namespace kvx;

extern "C" {

int kvx_store_kvcache_q4(int32_t device, int32_t dtype, const void* key_dev, const void* value_dev,
                         int64_t key_token_stride, int64_t value_token_stride, void* k_cache_dev, void* v_cache_dev,
                         int64_t cache_block_stride, const int64_t* slot_mapping_dev, int64_t num_tokens,
                         int64_t num_blocks, int32_t block_size, int32_t kv_heads, int32_t head_dim, float k_scale,
                         float v_scale, int32_t* status_dev, void* stream) {
    return q4_launch(true, device, dtype, key_dev, value_dev, key_token_stride, value_token_stride, k_cache_dev,
                     v_cache_dev, cache_block_stride, slot_mapping_dev, num_tokens, num_blocks, block_size, kv_heads,
                     head_dim, k_scale, v_scale, status_dev, stream);
}

int kvx_load_kvcache_q4(int32_t device, int32_t dtype, void* key_dev, void* value_dev, int64_t key_token_stride,
                        int64_t value_token_stride, const void* k_cache_dev, const void* v_cache_dev,
                        int64_t cache_block_stride, const int64_t* slot_mapping_dev, int64_t num_tokens,
                        int64_t num_blocks, int32_t block_size, int32_t kv_heads, int32_t head_dim, float k_scale,
                        float v_scale, int32_t* status_dev, void* stream) {
    return q4_launch(false, device, dtype, key_dev, value_dev, key_token_stride, value_token_stride, k_cache_dev,
                     v_cache_dev, cache_block_stride, slot_mapping_dev, num_tokens, num_blocks, block_size, kv_heads,
                     head_dim, k_scale, v_scale, status_dev, stream);
}

}  // extern "C"
