// C ABI of a serving step's operators: pages and slots of the cache, attention over the cached latents.
// Declarations: include/pypto_amd_sfa.h.
#include <hip/hip_runtime.h>

#include <cmath>

#include "capi_error.h"
#include "common.h"
#include "pypto_amd_sfa.h"
#include "serving_ops.h"

namespace {

using pto::cu_count;
using pto::fail;

constexpr int64_t MOST_TOKENS = 1ll << 30;
constexpr int PACKED_PITCH = 656;

bool aligned(const void *p, const uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int table_check(const char *op, const int64_t b, const int64_t maxblk, const int64_t bs)
{
    if (b < 1 || b > (1ll << 24)) return fail(PTO_E_INVALID_ARG, "%s: b out of range", op);
    if (bs < 1 || bs > (1ll << 30) || maxblk < 1 || maxblk > (1ll << 30))
        return fail(PTO_E_INVALID_ARG, "%s: block_size and max_blocknum_perbatch must be in [1, 2^30]", op);
    if (b * maxblk > 0x7fffffffll) return fail(PTO_E_INVALID_ARG, "%s: a block table holds at most 2^31 - 1 entries", op);
    return PTO_OK;
}

int latent_check(const PtoLatentAttentionArgs *a)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "latent_attention: args is NULL");
    const int rc = table_check("latent_attention", a->b, a->max_blocknum_perbatch, a->block_size);
    if (rc != PTO_OK) return rc;
    if (a->total_q < 0 || a->total_q > MOST_TOKENS || a->heads < 1 || a->heads > 65536 || a->total_q * a->heads > 0x7fff0000ll)
        return fail(PTO_E_INVALID_ARG, "latent_attention: total_q or heads out of range");
    static_assert(pto::LA_MOST_KEYS == 0x7fffffff - 15);
    if (a->max_blocknum_perbatch * a->block_size > pto::LA_MOST_KEYS)
        return fail(PTO_E_INVALID_ARG, "latent_attention: a sequence of the block table holds at most 2^31 - 16 keys");
    if (a->window < 0 || a->window > MOST_TOKENS || a->sinks < 0 || a->sinks > MOST_TOKENS)
        return fail(PTO_E_INVALID_ARG, "latent_attention: window and sinks must be in [0, 2^30]");
    if (a->sinks > 0 && a->window == 0) return fail(PTO_E_INVALID_ARG, "latent_attention: sinks go with a window");
    if (a->tree_mask && a->window > 0) return fail(PTO_E_INVALID_ARG, "latent_attention: a tree mask and a window exclude one another");
    if (a->tree_mask && (a->mask_words < 1 || a->mask_words > pto::SLOTS_MAX_WORDS))
        return fail(PTO_E_INVALID_ARG, "latent_attention: mask_words must be in [1, %d]", pto::SLOTS_MAX_WORDS);
    if (!std::isfinite(a->softmax_scale) || !std::isfinite(a->softmax_scale * 1.4426950408889634f))
        return fail(PTO_E_INVALID_ARG, "latent_attention: softmax_scale is not finite");
    return PTO_OK;
}

// A form's launch: how its row tiles may be divided, and the memory for their pieces.
struct LatentForm {
    int most_tiles, row_tiles, groups, by_tile, entries;
    size_t o_bytes, ml_bytes, join_bytes;
    size_t bytes() const { return o_bytes + ml_bytes + join_bytes; }
};
struct LatentPlan {
    bool narrow, wide;
    LatentForm form[2];                   // of 64 rows, of 128
    size_t bytes, flag;                   // of the workspace; where the word is that says which form it was
};

// The device divides the work, since lengths are there.  Here only as many workgroups as there can be pieces of LA_LEAST units, one to a
// compute unit at most (a workgroup's LDS is most of one's), and memory for two pieces of each.
LatentForm latent_form(const PtoLatentAttentionArgs *a, const int rows, const long long cus)
{
    LatentForm f{};
    const long long row_tiles = a->total_q * a->heads / rows + (a->b < a->total_q ? a->b : a->total_q);          // at most
    long long tiles = (a->max_blocknum_perbatch * a->block_size + pto::LA_KEYS - 1) / pto::LA_KEYS;
    if (a->window > 0) {
        // of a row tile's tokens, the window of the first to the last one's last key, and the first keys
        const long long reach = a->window + (rows - 2) / a->heads + 1;
        const long long w = (a->sinks + pto::LA_KEYS - 1) / pto::LA_KEYS + (reach + pto::LA_KEYS - 1) / pto::LA_KEYS + 1;
        tiles = w < tiles ? w : tiles;
    }
    f.most_tiles = (int)tiles;
    f.row_tiles = (int)row_tiles;
    const double pieces = (double)row_tiles * (double)(tiles + pto::LA_OPEN) / pto::LA_LEAST;
    const long long groups = pieces < (double)cus ? (long long)pieces + 1 : cus;
    f.groups = (int)((groups + 7) / 8 * 8);
    f.by_tile = row_tiles <= f.groups;
    f.entries = (int)(f.by_tile ? (row_tiles > 0 ? row_tiles : 1) : f.groups);
    f.o_bytes = (size_t)2 * f.groups * rows * 512 * sizeof(float);
    f.ml_bytes = (size_t)2 * f.groups * rows * 2 * sizeof(float);
    f.join_bytes = (size_t)f.entries * 4 * sizeof(int32_t);
    return f;
}

// 128 rows to a workgroup read a tile of keys half as often, for twice the bytes to a piece and a longer beginning.  What that comes to hangs on lengths:
// on tiles to a compute unit, which 128 rows want many of, or on row tiles so many that few are cut into pieces, and on how much of 128 rows sequences leave empty
// (no more than an eighth above what they leave of 64).  The table's width says nothing of them: in a captured step it is that of the longest context there
// can be.  So where its width leaves both open, both forms are launched and the first one finds from the lengths which of them returns at once; that
// costs 3 to 5 us.  64 rows and 128, us, of 128 heads where not said otherwise:
//   single tokens: 1 over 500 keys 19.3 and 24.9, over 30000 (7 tiles of 64 rows to a compute unit) 36.5 and 46.7, over 130000 (32) 72 and 76, over 500000 (122)
//   222 and 197; 32 over 2052 (16) 47 and 54, over 8000 (62) 110 and 109, over 16000 (125) 207 and 190; 128 over 500 (16) 42 and 58, over 2000 (63) 105 and 112
//   4 of 30 tokens over 200 keys (7) 36 and 42, over 1000 (30) 71.4 and 69.9, over 2030 (60) 114 and 105
//   many row tiles: 208 single tokens over 60, 300, 1000 keys 32.7, 61.8, 114 and 29.8, 58.7, 118; 256: 35, 59, 121 and 31, 49, 100; 512: 62, 111, 256 and 52, 89, 212;
//   5 of 40 tokens over 60, 300, 1000 keys 30.5, 56.6, 106 and 27.2, 53.5, 100; 160 single tokens 30.5, 53, 95 and 28, 60, 93
//   rows that are padded: 150 of 9 tokens of 16 heads over 60 keys 29.4 and 40, over 1000 119 and 135; 16 of 4 tokens, 40 heads, over 20000 183 and 197
constexpr long long WIDE_TILES = 40;      // of 64 rows, to a compute unit
long long wide_row_tiles(const long long cus) { return 3 * cus / 2; }

LatentPlan latent_plan(const PtoLatentAttentionArgs *a)
{
    LatentPlan pl{};
    const long long cus = cu_count() > 0 ? cu_count() : 256, rows = a->total_q * a->heads;
    pl.form[0] = latent_form(a, pto::LA_ROWS, cus);
    pl.form[1] = latent_form(a, pto::LA_WIDE_ROWS, cus);
    const bool many = rows >= wide_row_tiles(cus) * pto::LA_ROWS;
    const bool unpadded = a->heads % pto::LA_WIDE_ROWS == 0 || rows >= 1024 * a->b;
    pl.wide = rows >= 96 * a->b && (many || (double)rows * (double)pl.form[0].most_tiles >= (double)(WIDE_TILES * cus * pto::LA_ROWS));
    pl.narrow = !pl.wide || !many || !unpadded;
    for (int i = 0; i < 2; ++i)
        if (i ? pl.wide : pl.narrow) pl.bytes = pl.form[i].bytes() > pl.bytes ? pl.form[i].bytes() : pl.bytes;
    if (pl.narrow && pl.wide) {
        pl.flag = (pl.bytes + 15) / 16 * 16;
        pl.bytes = pl.flag + 16;
    }
    return pl;
}

}  // namespace

extern "C" {

int pto_cache_pages_launch(const PtoCachePagesArgs *a, void *hip_stream)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "cache_pages: args is NULL");
    const int rc = table_check("cache_pages", a->b, a->max_blocknum_perbatch, a->block_size);
    if (rc != PTO_OK) return rc;
    if (a->room < 0 || a->room > 0x7fffffffll) return fail(PTO_E_INVALID_ARG, "cache_pages: room out of range");
    if (!a->lens_before || !a->lens_after || !a->block_table || !a->free_count || !a->free_left || (a->room > 0 && !a->free_pages))
        return fail(PTO_E_INVALID_ARG, "cache_pages: a tensor pointer is NULL");
    if (!aligned(a->lens_before, 4) || !aligned(a->lens_after, 4) || !aligned(a->block_table, 4) || !aligned(a->free_pages, 4) || !aligned(a->free_count, 4) ||
        !aligned(a->free_left, 4))
        return fail(PTO_E_INVALID_ARG, "cache_pages: pointers must be aligned to their element size");
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "cache_pages: no usable device is current");
    pto::CachePagesParams p{};
    p.before = a->lens_before;
    p.after = a->lens_after;
    p.bt = a->block_table;
    p.stack = a->free_pages;
    p.count = a->free_count;
    p.left = a->free_left;
    p.room = a->room;
    p.B = (int)a->b;
    p.maxblk = (int)a->max_blocknum_perbatch;
    p.bs = (int)a->block_size;
    const hipError_t e = pto::cache_pages_launch(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "cache_pages: launch failed: %s", hipGetErrorString(e));
    return PTO_OK;
}

int pto_cache_slots_launch(const PtoCacheSlotsArgs *a, void *hip_stream)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "cache_slots: args is NULL");
    const int rc = table_check("cache_slots", a->b, a->max_blocknum_perbatch, a->block_size);
    if (rc != PTO_OK) return rc;
    if (a->t < 0 || a->t > MOST_TOKENS) return fail(PTO_E_INVALID_ARG, "cache_slots: t out of range");
    if (!a->parents != !a->tree_mask && a->t > 0) return fail(PTO_E_INVALID_ARG, "cache_slots: parents and tree_mask come together");
    if (a->tree_mask && (a->mask_words < 1 || a->mask_words > pto::SLOTS_MAX_WORDS))
        return fail(PTO_E_INVALID_ARG, "cache_slots: mask_words must be in [1, %d]", pto::SLOTS_MAX_WORDS);
    if (!a->query_lens || !a->seq_lens || !a->block_table || !a->cu_seqlens_q || (a->t > 0 && (!a->positions || !a->cache_index)))
        return fail(PTO_E_INVALID_ARG, "cache_slots: a tensor pointer is NULL");
    if (!aligned(a->query_lens, 4) || !aligned(a->seq_lens, 4) || !aligned(a->block_table, 4) || !aligned(a->cu_seqlens_q, 4) || !aligned(a->cu_seqlens_k, 4) ||
        !aligned(a->positions, 8) || !aligned(a->cache_index, 8) || !aligned(a->parents, 4) || !aligned(a->tree_mask, 8))
        return fail(PTO_E_INVALID_ARG, "cache_slots: pointers must be aligned to their element size");
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "cache_slots: no usable device is current");
    pto::CacheSlotsParams p{};
    p.new_lens = a->query_lens;
    p.all_lens = a->seq_lens;
    p.bt = a->block_table;
    p.cu_q = a->cu_seqlens_q;
    p.cu_k = a->cu_seqlens_k;
    p.positions = reinterpret_cast<long long *>(a->positions);
    p.slots = reinterpret_cast<long long *>(a->cache_index);
    p.parents = a->parents;
    p.mask = reinterpret_cast<unsigned long long *>(a->tree_mask);
    p.T = a->t;
    p.B = (int)a->b;
    p.maxblk = (int)a->max_blocknum_perbatch;
    p.bs = (int)a->block_size;
    p.words = (int)a->mask_words;
    p.cus = cu_count();
    const hipError_t e = pto::cache_slots_launch(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "cache_slots: launch failed: %s", hipGetErrorString(e));
    return PTO_OK;
}

int pto_latent_attention_workspace_bytes(const PtoLatentAttentionArgs *a, size_t *bytes)
{
    if (!bytes) return fail(PTO_E_INVALID_ARG, "latent_attention: bytes is NULL");
    const int rc = latent_check(a);
    if (rc != PTO_OK) return rc;
    *bytes = latent_plan(a).bytes;
    return PTO_OK;
}

int pto_latent_attention_launch(const PtoLatentAttentionArgs *a, void *hip_stream)
{
    const int rc = latent_check(a);
    if (rc != PTO_OK || a->total_q == 0) return rc;
    const bool packed = a->packed != 0;
    if (a->cache_rows < 1 || a->cache_rows > 0x7fffffffll) return fail(PTO_E_INVALID_ARG, "latent_attention: cache_rows out of range");
    if (!a->nope || (packed ? a->rope_cache || a->scales : !a->rope_cache || !a->scales))
        return fail(PTO_E_INVALID_ARG, "latent_attention: a cache is three arrays, or one packed array and two NULL pointers");
    if (!a->query_nope || !a->query_rope || !a->out || !a->block_table || !a->cu_seqlens_q || !a->seq_lens)
        return fail(PTO_E_INVALID_ARG, "latent_attention: a tensor pointer is NULL");
    if (!aligned(a->nope, 16) || !aligned(a->rope_cache, 16) || !aligned(a->scales, 16))
        return fail(PTO_E_INVALID_ARG, "latent_attention: cache pointers must be 16-byte aligned");
    if (!aligned(a->query_nope, 16) || !aligned(a->query_rope, 16) || a->query_nope_stride_t % 8 != 0 || a->query_nope_stride_h % 8 != 0 ||
        a->query_rope_stride_t % 8 != 0 || a->query_rope_stride_h % 8 != 0)
        return fail(PTO_E_INVALID_ARG, "latent_attention: queries must be 16-byte aligned, their strides multiples of 8 elements");
    if (!aligned(a->out, 2) || !aligned(a->lse, 4) || !aligned(a->block_table, 4) || !aligned(a->cu_seqlens_q, 4) || !aligned(a->seq_lens, 4) ||
        !aligned(a->tree_mask, 8))
        return fail(PTO_E_INVALID_ARG, "latent_attention: pointers must be aligned to their element size");
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "latent_attention: no usable device is current");
    const LatentPlan pl = latent_plan(a);
    if (!a->workspace || a->workspace_bytes < pl.bytes)
        return fail(PTO_E_WORKSPACE, "latent_attention: workspace of %zu bytes required, %zu given", pl.bytes, a->workspace ? a->workspace_bytes : (size_t)0);
    if (!aligned(a->workspace, 16)) return fail(PTO_E_INVALID_ARG, "latent_attention: the workspace must be 16-byte aligned");

    pto::LaParams p{};
    p.q = static_cast<const uint16_t *>(a->query_nope);
    p.qr = static_cast<const uint16_t *>(a->query_rope);
    p.q_t = a->query_nope_stride_t, p.q_h = a->query_nope_stride_h;
    p.qr_t = a->query_rope_stride_t, p.qr_h = a->query_rope_stride_h;
    p.o_t = a->out_stride_t, p.o_h = a->out_stride_h;
    p.cache.nope = static_cast<uint8_t *>(const_cast<void *>(a->nope));
    p.cache.rope = packed ? p.cache.nope + 512 : static_cast<uint8_t *>(const_cast<void *>(a->rope_cache));
    p.cache.scale = packed ? p.cache.nope + 640 : static_cast<uint8_t *>(const_cast<void *>(a->scales));
    p.cache.nope_pitch = packed ? PACKED_PITCH : 512;
    p.cache.rope_pitch = packed ? PACKED_PITCH : 128;
    p.cache.scale_pitch = packed ? PACKED_PITCH : 16;
    p.cache.rows = a->cache_rows;
    p.bt = a->block_table;
    p.cu_q = a->cu_seqlens_q;
    p.lens = a->seq_lens;
    p.mask = reinterpret_cast<const unsigned long long *>(a->tree_mask);
    p.out = static_cast<uint16_t *>(a->out);
    p.lse = a->lse;
    p.total_q = a->total_q;
    p.B = (int)a->b;
    p.maxblk = (int)a->max_blocknum_perbatch;
    p.bs = (int)a->block_size;
    p.heads = (int)a->heads;
    p.words = a->tree_mask ? (int)a->mask_words : 0;
    p.window = (int)a->window;
    p.sinks = (int)a->sinks;
    p.most_keys = (int)(a->max_blocknum_perbatch * a->block_size);
    p.of_heads = pto::divisor_of((uint32_t)a->heads);
    p.of_bs = pto::divisor_of((uint32_t)a->block_size);
    p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
    char *const ws = static_cast<char *>(a->workspace);
    if (pl.narrow && pl.wide) p.form = reinterpret_cast<int32_t *>(ws + pl.flag), p.wide_tiles = WIDE_TILES * cu_count(), p.wide_row_tiles = wide_row_tiles(cu_count());
    pto::LaParams of[2] = {p, p};
    for (int i = 0; i < 2; ++i) {
        const LatentForm &f = pl.form[i];
        const int threads = i ? pto::LA_WIDE_THREADS : pto::LA_THREADS;
        of[i].part_o = reinterpret_cast<float *>(ws);
        of[i].part_ml = reinterpret_cast<float *>(ws + f.o_bytes);
        of[i].joins = reinterpret_cast<int32_t *>(ws + f.o_bytes + f.ml_bytes);
        of[i].most_tiles = f.most_tiles;
        of[i].per_entry = (int)((a->b + threads - 1) / threads);
        of[i].seq_entries = (int)((a->b + of[i].per_entry - 1) / of[i].per_entry);
        of[i].groups = f.groups;
        of[i].most_row_tiles = f.row_tiles;
        of[i].by_tile = f.by_tile;
        of[i].entries = f.entries;
    }
    const hipError_t e = pto::latent_attention_launch(pl.narrow ? &of[0] : nullptr, pl.wide ? &of[1] : nullptr, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "latent_attention: launch failed: %s", hipGetErrorString(e));
    return PTO_OK;
}

}  // extern "C"
