// Paged attention, host side: argument checks, the choice between the two
// kernels and the number of splits of the key axis.

#include <algorithm>
#include <climits>
#include <cmath>

#include "kvx.h"
#include "kvx_attn.cuh"
#include "kvx_host.h"

namespace kvx {

// Splits of the key axis. Figures: us a call, bf16, 32 heads on 8 of 128 unless stated, `a x b` = a sequences of b keys.
// CTAs of the split kernel to aim for, in fills of the GPU (more: an even end; fewer: less to join). 1 / 2 / 4 / 8: 4 x 50000
// 150/146/147/149; 16 x 6000 86/85/88/90; 100 x 3000 205/205/205/215; 4-bit 8 x 8000 31/34/34/34, 100 x 3000 96/96/95/108.
constexpr int kWaves = 4;
// Keys of a split, at least. 128 / 256 / 512 / 1024 / 2048: 2 x 700 12/14/16/16/16; 8 x 1500 27/25/21/27/27; 16 x 6000
// 88/88/88/94/86; 4-bit 2 x 700 11/12/13/13/13, 4 x 1500 14/14/14/19/19, 8 x 8000 40/39/34/31/33.
constexpr int kMinKeys = 512;
// Key tiles (of 128) of a split of the tile kernel, at least. 1 / 2 / 4 / 8: 64 tokens on 7936 keys 33/33/35/43, 2 x 40 tokens
// on 2960 31/31/32/40, 32 on 968 22/25/27/31; 4-bit 64 on 7936 38/37/39/47.
constexpr int kMinTiles = 4;
// Rows of a sequence and kv head (tokens x group heads) up to which the split kernel is taken. Split against tile
// kernel, us, bf16, 8 kv heads of 128, 12, 16 and 24 rows. 16-bit cache, 32 sequences of 2000 keys: 82/90, 85/90, 97/90; 256 of
// 600: 149/182, 154/182, 184/182; 4 of 30000: 116/157, 118/157, 130/157. 4-bit cache: 63/89, 67/89, 87/89; 121/207, 129/208,
// 172/207; 81/151, 83/151, 108/151 (at 32 rows, in two passes of the split kernel: 122/99; 241/232; 146/161).
constexpr int kFewRows16 = 16;
constexpr int kFewRows4 = 24;
constexpr int kTileRows = 256;          // rows of an item of the tile kernel

struct AttnPlan {
    bool tile;          // tile kernel, else split kernel
    int nt;             // row tiles of 8 (split kernel)
    int tile_tokens;
    int tile_slots;
    int splits;
    int min_tiles;      // key tiles of a split, at least
    uint64_t workspace;
};

static int check_args(const kvx_attention* a) {
    if (a == nullptr) return fail(KVX_EINVAL, "args is NULL");
    if (a->reserved[0] != 0 || a->reserved[1] != 0) return fail(KVX_EINVAL, "reserved must be 0");
    if (a->dtype != 0 && a->dtype != 1) return fail(KVX_EINVAL, "dtype must be 0 (bf16) or 1 (fp16)");
    if (a->cache_bits != 16 && a->cache_bits != 4) return fail(KVX_EINVAL, "cache_bits must be 16 or 4");
    if (a->head_dim != 64 && a->head_dim != 128) return fail(KVX_EINVAL, "head_dim must be 64 or 128 (got %d)", a->head_dim);
    if (a->num_tokens < 0 || a->num_seqs < 0) return fail(KVX_EINVAL, "negative token or sequence count");
    if (static_cast<int64_t>(a->num_tokens) + a->num_seqs > INT_MAX)     // slots of items are counted in 32 bits
        return fail(KVX_EINVAL, "num_tokens + num_seqs is beyond 2^31 - 1");
    if (a->num_heads <= 0 || a->num_kv_heads <= 0 || a->num_heads % a->num_kv_heads != 0)
        return fail(KVX_EINVAL, "num_heads (%d) must be a multiple of num_kv_heads (%d)", a->num_heads, a->num_kv_heads);
    if (a->num_kv_heads > 65535) return fail(KVX_EINVAL, "num_kv_heads must be at most 65535");
    if (a->num_heads / a->num_kv_heads > kTileRows)
        return fail(KVX_EINVAL, "at most %d query heads per kv head", kTileRows);
    if (a->block_size <= 0) return fail(KVX_EINVAL, "block_size must be > 0");
    if (a->cache_bits == 4 && a->block_size % 16 != 0)
        return fail(KVX_EINVAL, "block_size of a 4-bit cache must be a multiple of 16");
    // The kernels index within a (page, head) of a 4-bit cache in 32 bits, as the store does.
    if (a->cache_bits == 4 && static_cast<int64_t>(a->block_size) * a->head_dim > INT_MAX / 2)
        return fail(KVX_EINVAL, "block_size * head_dim is too large");
    if (a->table_width < 0) return fail(KVX_EINVAL, "table_width must be >= 0");
    if (static_cast<int64_t>(a->table_width) * a->block_size > INT_MAX - 1024)
        return fail(KVX_EINVAL, "table_width * block_size is beyond 2^31 - 1025 keys");
    if (a->num_blocks <= 0) return fail(KVX_EINVAL, "num_blocks must be > 0");
    if (a->window < 0 || a->sinks < 0) return fail(KVX_EINVAL, "window and sinks must be >= 0");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(KVX_EINVAL, "scale must be positive and finite");
    if (!power_of_two(a->k_scale) || !power_of_two(a->v_scale))
        return fail(KVX_EINVAL, "k_scale and v_scale must be powers of two in [2^-64, 2^63]");
    if (a->cache_bits == 16 && (a->k_scale != 1.f || a->v_scale != 1.f))
        return fail(KVX_EINVAL, "k_scale and v_scale belong to 4-bit caches");
    const float logits = a->scale * 1.44269504088896340736f * a->k_scale;
    if (!(logits >= 1.17549435e-38f) || !std::isfinite(logits))
        return fail(KVX_EINVAL, "scale * k_scale is outside the range of fp32");
    if (a->cu_seqlens_q == 0 && a->num_tokens != a->num_seqs)
        return fail(KVX_EINVAL, "without cu_seqlens_q every sequence has one token (%d tokens, %d sequences)",
                    a->num_tokens, a->num_seqs);
    return KVX_OK;
}

// What fills the GPU: an SM takes 2 CTAs of the split kernel on a 16-bit cache (shared memory), 4 on a 4-bit one with
// one row tile, 2 with more (registers); the tile kernel has one.
static AttnPlan plan_of(const kvx_attention* a, int sms) {
    AttnPlan pl{};
    const int group = a->num_heads / a->num_kv_heads;
    const int64_t tokens = a->num_tokens, seqs = std::max(1, a->num_seqs);
    const int64_t avg = (tokens + seqs - 1) / seqs;
    pl.tile = avg * group > (a->cache_bits == 4 ? kFewRows4 : kFewRows16);
    int keys_per_tile, fill;
    if (pl.tile) {
        // Sequences of few rows: items of one row tile, the other half of the kernel rests.
        pl.tile_tokens = (avg * group <= kTileRows / 2 ? kTileRows / 2 : kTileRows) / group;
        keys_per_tile = 128;
        fill = sms;
        pl.min_tiles = kMinTiles;
    } else {
        // One pass over the keys for a sequence of average length. (A pass costs what it reads and widens, and a row tile less
        // than that: two passes of fewer rows never pay.)
        pl.nt = static_cast<int>((avg * group + 7) / 8);
        pl.tile_tokens = a->cu_seqlens_q ? 8 * pl.nt / group : 1;
        const bool q4 = a->cache_bits == 4;
        keys_per_tile = q4 && pl.nt < 3 ? 128 : 64;
        fill = sms * (q4 && pl.nt == 1 ? 4 : 2) * kWaves;
        pl.min_tiles = kMinKeys / keys_per_tile;
    }
    pl.tile_slots = static_cast<int>(a->cu_seqlens_q ? tokens / pl.tile_tokens + a->num_seqs : a->num_seqs);
    const int64_t items = std::max<int64_t>(seqs, (tokens + pl.tile_tokens - 1) / pl.tile_tokens) * a->num_kv_heads;
    // The most keys that a sequence can have to read, from what the host knows.
    int64_t keys = static_cast<int64_t>(a->table_width) * a->block_size;
    if (a->window > 0)
        keys = std::min(keys, static_cast<int64_t>(a->window) + a->sinks + pl.tile_tokens + 2 * keys_per_tile);
    const int64_t tiles = (keys + keys_per_tile - 1) / keys_per_tile;
    int64_t splits = fill / std::max<int64_t>(1, items);
    splits = std::min(splits, tiles / pl.min_tiles);
    pl.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(splits, kMaxSplits)));
    if (pl.splits > 1)
        pl.workspace = static_cast<uint64_t>(tokens) * a->num_heads * pl.splits * (a->head_dim + 2) * 4;
    return pl;
}

}  // namespace kvx

using namespace kvx;

extern "C" {

int kvx_attention_workspace(int32_t device, const kvx_attention* args, uint64_t* bytes_out) {
    if (bytes_out == nullptr) return fail(KVX_EINVAL, "bytes_out is NULL");
    int rc = check_args(args);
    if (rc != KVX_OK) return rc;
    int sms = 0;
    rc = sm_count(device, &sms);
    if (rc != KVX_OK) return rc;
    *bytes_out = args->num_tokens == 0 ? 0 : plan_of(args, sms).workspace;
    return KVX_OK;
}

int kvx_paged_attention(int32_t device, const kvx_attention* args, void* workspace_dev, uint64_t workspace_bytes,
                        int32_t* status_dev, void* stream) {
    int rc = check_args(args);
    if (rc != KVX_OK) return rc;
    const kvx_attention& a = *args;
    if (status_dev == nullptr) return fail(KVX_EINVAL, "status_dev is NULL");
    if (a.num_tokens == 0 || a.num_seqs == 0) return KVX_OK;
    if (!a.query || !a.out || !a.k_cache || !a.v_cache || !a.context_lens || (!a.block_tables && a.table_width > 0))
        return fail(KVX_EINVAL, "NULL tensor pointer");
    uint64_t bits = a.query | a.out | a.k_cache | a.v_cache | static_cast<uint64_t>(a.query_token_stride) |
                    static_cast<uint64_t>(a.query_head_stride) | static_cast<uint64_t>(a.out_token_stride) |
                    static_cast<uint64_t>(a.out_head_stride) | static_cast<uint64_t>(a.cache_block_stride) |
                    reinterpret_cast<uint64_t>(workspace_dev);
    if (a.cache_bits == 16)
        bits |= static_cast<uint64_t>(a.cache_slot_stride) | static_cast<uint64_t>(a.cache_head_stride);
    if (bits & 15) return fail(KVX_EINVAL, "addresses and strides must be multiples of 16 bytes");
    if (reinterpret_cast<uint64_t>(workspace_dev) & 31) return fail(KVX_EINVAL, "workspace_dev must be 32-byte aligned");
    int sms = 0;
    rc = sm_count(device, &sms);
    if (rc != KVX_OK) return rc;
    const AttnPlan pl = plan_of(args, sms);
    if (pl.workspace > 0 && (workspace_dev == nullptr || workspace_bytes < pl.workspace))
        return fail(KVX_EINVAL, "workspace of %llu bytes needed, got %llu", static_cast<unsigned long long>(pl.workspace),
                    static_cast<unsigned long long>(workspace_bytes));
    AttnParams p{};
    p.q = reinterpret_cast<const char*>(a.query);
    p.out = reinterpret_cast<char*>(a.out);
    p.k = reinterpret_cast<const char*>(a.k_cache);
    p.v = reinterpret_cast<const char*>(a.v_cache);
    p.q_token_stride = a.query_token_stride;
    p.q_head_stride = a.query_head_stride;
    p.o_token_stride = a.out_token_stride;
    p.o_head_stride = a.out_head_stride;
    p.block_stride = a.cache_block_stride;
    p.slot_stride = a.cache_slot_stride;
    p.head_stride = a.cache_bits == 4 ? static_cast<int64_t>(a.block_size) * (a.head_dim / 16 * 9) : a.cache_head_stride;
    p.num_blocks = a.num_blocks;
    p.table = reinterpret_cast<const int32_t*>(a.block_tables);
    p.table_stride = a.table_stride;
    p.ctx = reinterpret_cast<const int32_t*>(a.context_lens);
    p.cu = reinterpret_cast<const int32_t*>(a.cu_seqlens_q);
    p.status = status_dev;
    p.scale_log2 = a.scale * 1.44269504088896340736f * a.k_scale;
    p.out_scale = a.v_scale;
    p.table_width = a.table_width;
    p.block_size = a.block_size;
    p.block_shift = -1;
    if ((a.block_size & (a.block_size - 1)) == 0)
        for (p.block_shift = 0; (1 << p.block_shift) < a.block_size;) ++p.block_shift;
    p.num_seqs = a.num_seqs;
    p.num_tokens = a.num_tokens;
    p.heads = a.num_heads;
    p.kv_heads = a.num_kv_heads;
    p.group = a.num_heads / a.num_kv_heads;
    p.window = a.window > 0 ? a.window : INT_MAX;
    p.sinks = a.sinks;
    p.splits = pl.splits;
    p.min_tiles = pl.min_tiles;
    p.tile_tokens = pl.tile_tokens;
    p.tile_slots = pl.tile_slots;
    p.out_wide = ((a.out | static_cast<uint64_t>(a.out_token_stride) | static_cast<uint64_t>(a.out_head_stride)) & 31) == 0;
    if (pl.splits > 1) {
        p.ws_o = static_cast<float*>(workspace_dev);
        p.ws_ml = p.ws_o + static_cast<int64_t>(a.num_tokens) * a.num_heads * pl.splits * a.head_dim;
    }
    if (pl.splits > 1 && static_cast<int64_t>(a.num_tokens) * a.num_heads > INT_MAX)
        return fail(KVX_EINVAL, "num_tokens * num_heads is beyond 2^31");
    KVX_DEVICE_GUARD(device);
    const auto st = static_cast<cudaStream_t>(stream);
    const bool q4 = a.cache_bits == 4;
    rc = pl.tile ? launch_attn_tile(p, a.head_dim, a.dtype, q4, device, sms, st)
                 : launch_attn_split(p, a.head_dim, a.dtype, q4, pl.nt, device, st);
    if (rc == KVX_OK && pl.splits > 1) rc = launch_attn_join(p, a.head_dim, a.dtype, st);
    if (rc != KVX_OK) cudaGetLastError();
    return rc;
}

}  // extern "C"
