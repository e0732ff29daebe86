// C ABI of the operators around a prompt: argument validation, workspace sizing, launch plans.
// Declarations: include/pypto_amd_sfa.h.
#include <hip/hip_runtime.h>

#include <cmath>

#include "capi_error.h"
#include "common.h"
#include "prompt_ops.h"
#include "pypto_amd_sfa.h"

namespace {

using pto::cu_count;
using pto::fail;

constexpr int64_t MOST_TOKENS = 1ll << 30;
constexpr int PACKED_PITCH = 656;

bool aligned(const void *p, const uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool dtype_known(const int32_t d) { return d == PTO_DT_FP16 || d == PTO_DT_FP32 || d == PTO_DT_BF16; }
uintptr_t element(const int32_t d) { return d == PTO_DT_FP32 ? 4 : 2; }

int tables_check(const PtoRotaryTablesArgs *a)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "rotary_tables: args is NULL");
    if (a->t < 0 || a->t > MOST_TOKENS) return fail(PTO_E_INVALID_ARG, "rotary_tables: t out of range");
    if (a->pairs < 4 || a->pairs % 4 != 0 || a->pairs > pto::ROT_MAX_PAIRS)
        return fail(PTO_E_INVALID_ARG, "rotary_tables: pairs must be a multiple of 4, up to %d (got %lld)", pto::ROT_MAX_PAIRS, (long long)a->pairs);
    if (!dtype_known(a->dtype)) return fail(PTO_E_INVALID_ARG, "rotary_tables: unknown dtype code %d", a->dtype);
    if (!std::isfinite(a->factor)) return fail(PTO_E_INVALID_ARG, "rotary_tables: factor is not finite");
    if (a->t == 0) return PTO_OK;
    if (!a->positions || !a->frequencies || !a->cos || !a->sin) return fail(PTO_E_INVALID_ARG, "rotary_tables: a tensor pointer is NULL");
    if (!aligned(a->positions, a->positions_int64 ? 8 : 4) || !aligned(a->frequencies, 8) || !aligned(a->cos, element(a->dtype)) ||
        !aligned(a->sin, element(a->dtype)))
        return fail(PTO_E_INVALID_ARG, "rotary_tables: pointers must be aligned to their element size");
    return PTO_OK;
}

int rotary_side(const PtoRotaryTensor &t, const char *name, const int64_t pairs, const int32_t dtype, pto::RotarySide &s)
{
    if (t.heads < 1 || t.heads > 65536 || t.dim < 1 || t.dim > 65536)
        return fail(PTO_E_INVALID_ARG, "rotary: %s: heads and dim must be in [1, 65536]", name);
    if (t.offset < 0 || t.offset + 2 * pairs > t.dim)
        return fail(PTO_E_INVALID_ARG, "rotary: %s: channels %lld .. %lld of %lld cannot turn", name, (long long)t.offset,
                    (long long)(t.offset + 2 * pairs - 1), (long long)t.dim);
    if (!t.in || !t.out) return fail(PTO_E_INVALID_ARG, "rotary: %s: a tensor pointer is NULL", name);
    if (!aligned(t.in, element(dtype)) || !aligned(t.out, element(dtype)))
        return fail(PTO_E_INVALID_ARG, "rotary: %s: pointers must be aligned to their element size", name);
    const bool in_place = t.in == t.out;
    if (in_place && (t.in_stride_t != t.out_stride_t || t.in_stride_h != t.out_stride_h))
        return fail(PTO_E_INVALID_ARG, "rotary: %s: in and out begin together but have different strides", name);
    s.in = t.in;
    s.out = t.out;
    s.heads = (int)t.heads;
    s.dim = (int)t.dim;
    s.offset = (int)t.offset;
    s.copies = !in_place && t.dim > 2 * pairs;
    s.in_t = t.in_stride_t;
    s.in_h = t.in_stride_h;
    s.out_t = t.out_stride_t;
    s.out_h = t.out_stride_h;
    return PTO_OK;
}

int cache_of(const char *op, const void *nope, const void *rope, const void *scales, const bool packed, const int64_t rows, pto::CacheRows &c)
{
    if (rows < 1 || rows > 0x7fffffffll) return fail(PTO_E_INVALID_ARG, "%s: cache_rows out of range", op);
    if (!nope || (packed ? rope || scales : !rope || !scales))
        return fail(PTO_E_INVALID_ARG, "%s: a cache is three arrays, or one packed array and two NULL pointers", op);
    if (!aligned(nope, 16) || !aligned(rope, 16) || !aligned(scales, 16))
        return fail(PTO_E_INVALID_ARG, "%s: cache pointers must be 16-byte aligned", op);
    c.nope = static_cast<uint8_t *>(const_cast<void *>(nope));
    c.rope = packed ? c.nope + 512 : static_cast<uint8_t *>(const_cast<void *>(rope));
    c.scale = packed ? c.nope + 640 : static_cast<uint8_t *>(const_cast<void *>(scales));
    c.nope_pitch = packed ? PACKED_PITCH : 512;
    c.rope_pitch = packed ? PACKED_PITCH : 128;
    c.scale_pitch = packed ? PACKED_PITCH : 16;
    c.rows = rows;
    return PTO_OK;
}

int attention_check(const char *op, const PtoPromptAttentionArgs *a)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "%s: args is NULL", op);
    if (a->b < 1 || a->b > (1ll << 24) || a->total_q < 0 || a->total_q > MOST_TOKENS || a->total_k < 0 || a->total_k > MOST_TOKENS)
        return fail(PTO_E_INVALID_ARG, "%s: b, total_q or total_k out of range", op);
    if (a->kv_heads < 1 || a->heads < 1 || a->heads > 65536 || a->heads % a->kv_heads != 0)
        return fail(PTO_E_INVALID_ARG, "%s: heads must be a multiple of kv_heads, up to 65536 (got %lld and %lld)", op, (long long)a->heads,
                    (long long)a->kv_heads);
    if (a->total_q * (a->heads / a->kv_heads) > 0x7fff0000ll)
        return fail(PTO_E_INVALID_ARG, "%s: total_q x heads of a group out of range", op);
    if (a->d != 64 && a->d != 128) return fail(PTO_E_INVALID_ARG, "%s: d must be 64 or 128 (got %lld)", op, (long long)a->d);
    if (!a->query_rope != !a->key_rope) return fail(PTO_E_INVALID_ARG, "%s: query_rope and key_rope come together", op);
    if (a->query_rope && a->d != 128) return fail(PTO_E_INVALID_ARG, "%s: rope parts go with d = 128", op);
    if (!std::isfinite(a->softmax_scale) || !std::isfinite(a->softmax_scale * 1.4426950408889634f))
        return fail(PTO_E_INVALID_ARG, "%s: softmax_scale is not finite", op);
    return PTO_OK;
}

struct PromptPlan {
    int splits, split_tiles, waves, most_tiles;
    long long workgroups;
    size_t o_bytes, ml_bytes;
};

// Eight waves to a workgroup or four.  Four leave room for a second workgroup on the compute unit, whose work stands in for one's waits at its
// beginning and end, and waste less on a short sequence; eight read a tile of keys half as often.  64 channels: four are never slower (3760
// causal tokens, 128/16 heads, 321 us with eight, 301 with four; 11 sequences of 72 to 243 tokens over 2100 keys, 128/32 heads, 214 and
// 185; 11 of 1 to 2 over 600, 128 heads, 83 and 51).  128 channels: four for fewer than 512 rows to a sequence and key head (6 sequences
// of 66 to 445 tokens over 1000 keys, 32 heads, 53 and 41; with rope parts 9 of 33 to 206 tokens, 128 heads, 68 and 61, 3 of 3 to 17
// over 2500 keys, 64/16 heads, 38 and 28), and for so few tiles that eight would fill half of the chip or less, unless there are many
// keys (412 tokens, 16/2 heads, 15.8 and 13.7; 2 of 369, 16/1 heads and rope parts, 17.7 and 15.4; but 5 of 74 to 535 over 6284 to 11824 keys,
// 8/4 heads and rope parts, 116 and 122).  For more eight (9 prompts of 65 to 1871 tokens, 64/8 heads, 166 and 176; 2 of 1841 and 2988, 32/8
// heads, 108 and 114).
//
// Dividing a call's keys.  The host knows how many rows, keys and sequences there are, not which sequence has how many, and takes them for
// dealt out evenly.  In microseconds: a workgroup starts and ends in `fixed`, takes `tile` for 64 keys, and partial results are written
// and read back by a launch of their own, `merge` and a tenth of a microsecond to a piece.  With s pieces to the longest row tile a launch
// takes the longest workgroup and then, for the rounds of the chip behind the first, the mean one; the cheapest s is taken if it saves a
// tenth (2 tokens over 6180 keys, 4 heads: 115 us in one piece, now 17; 294 over 4732, 8 heads: 92, now 28).  What is fixed is the
// length of a piece, so a sequence longer than the mean is divided into more.  Where the cheapest is one piece and the workgroups are few
// and very long, all sequences are divided, in pieces of half of the mean: one that is much longer would be there alone at the end (32
// sequences of 700 to 12000 keys, 8 key heads: 200 us, now 187).
// A launch has a workgroup for each row tile, or piece of one, that there can be, and the device starts the next as one ends; where that
// could be more than four for each compute unit, the workgroups of a divided launch take the pieces there are in turn.
constexpr size_t PA_MOST_PARTIALS = (size_t)256 << 20;

// A window bounds the tiles of any row tile: those of the first keys, those that the windows of its tokens reach over, and one more where these
// begin inside a tile.  The plan then takes a sequence for no longer.
PromptPlan attention_plan(const PtoPromptAttentionArgs *a, const int64_t window, const int64_t sinks)
{
    PromptPlan pl{};
    const long long cus = cu_count() > 0 ? cu_count() : 256;
    const long long rows = a->total_q * (a->heads / a->kv_heads);
    long long key_tiles = (a->total_k + pto::PA_KEYS - 1) / pto::PA_KEYS;                   // of one sequence, at most
    pl.splits = 1;
    const bool few = 2 * (rows / 256 + a->b) * a->kv_heads <= cus && a->total_k <= 4096 * a->b;
    pl.waves = a->d == 64 || rows < 512 * a->b || few ? 4 : 8;
    const int wg_rows = pl.waves * pto::PA_WAVE_ROWS;
    pl.most_tiles = 1 << 30;
    if (window > 0) {
        const long long reach = window + (wg_rows - 2) / (a->heads / a->kv_heads) + 1;
        pl.most_tiles = (int)((sinks + pto::PA_KEYS - 1) / pto::PA_KEYS + (reach + pto::PA_KEYS - 1) / pto::PA_KEYS + 1);
        key_tiles = key_tiles < pl.most_tiles ? key_tiles : pl.most_tiles;
    }
    const long long slots = pl.waves == 4 ? 2 * cus : cus;                                  // workgroups at a time
    const long long most_tiles = rows / wg_rows + a->b;                                     // of a key head
    pl.split_tiles = 1 << 24;
    pl.workgroups = most_tiles * a->kv_heads;

    const double seq_rows = (double)rows / a->b;
    const double items = (seq_rows <= wg_rows ? (double)a->b : (double)rows / wg_rows + (a->b > 1 ? 0.5 * a->b : 0.0)) * a->kv_heads;
    const double longest = std::fmin(std::ceil((double)a->total_k / a->b / pto::PA_KEYS), pl.most_tiles);
    const double mean = a->causal && a->total_k >= a->total_q ? std::fmin(((double)a->total_k - 0.5 * a->total_q) / a->b / pto::PA_KEYS, longest) : longest;
    if (items < 2.0 * slots && longest > 1.0) {
        const double fixed = 9.0, tile = a->d == 64 ? 1.1 : (a->query_rope ? 2.05 : 1.65);
        const double partial = (double)a->total_q * a->heads * (a->d + 2) * sizeof(float);
        const double merge = 4.0 + 3.0 * (double)a->total_q * a->heads / (32.0 * cus);
        auto pieces_of = [&](const long long len) { return (key_tiles + len - 1) / len; };
        auto cost = [&](const double s) {
            const double len = std::ceil(longest / s), rounds = std::ceil(std::ceil(items) * s / slots);
            return fixed + tile * len + (rounds - 1.0) * (fixed + tile * mean / s) + (s > 1.0 ? merge + s * (0.1 + partial * 0.5e-6) : 0.0);
        };
        double best = cost(1.0), s_best = 1.0;
        for (double s = 2.0; s <= longest && s <= pto::PA_MAX_SPLITS; s += 1.0)
            if (cost(s) < best) best = cost(s), s_best = s;
        if (best > 0.9 * cost(1.0)) s_best = 1.0;
        long long len = (long long)std::ceil(longest / s_best);
        if (s_best == 1.0) {
            const bool uneven = a->b > 1 && items <= 1.5 * slots;
            len = uneven && tile * longest >= 8.0 * fixed ? (len + 1) / 2 : key_tiles;
        }
        while (pieces_of(len) > pto::PA_MAX_SPLITS || (len < key_tiles && partial * (double)pieces_of(len) > (double)PA_MOST_PARTIALS)) len += (len + 3) / 4;
        if (pieces_of(len) > 1) {
            pl.splits = (int)pieces_of(len);
            pl.split_tiles = (int)len;
            const long long by_tiles = most_tiles * pl.splits, by_keys = window > 0 ? by_tiles : ((rows + wg_rows - 1) / wg_rows) * (key_tiles / len + a->b + 1);
            pl.workgroups = (by_tiles < by_keys ? by_tiles : by_keys) * a->kv_heads;
            if (pl.workgroups > 4 * slots) pl.workgroups = 4 * slots;
        }
    }
    pl.workgroups = (pl.workgroups + 7) / 8 * 8;
    if (pl.splits > 1) {
        pl.o_bytes = (size_t)a->total_q * a->heads * pl.splits * a->d * sizeof(float);
        pl.ml_bytes = (size_t)a->total_q * a->heads * pl.splits * 2 * sizeof(float);
    }
    return pl;
}

int attention_launch(const char *op, const PtoPromptAttentionArgs *a, const int64_t window, const int64_t sinks, void *hip_stream)
{
    if (a->total_q == 0) return PTO_OK;
    if (!a->query || !a->out || !a->cu_seqlens_q || !a->cu_seqlens_k || (a->total_k > 0 && (!a->key || !a->value)))
        return fail(PTO_E_INVALID_ARG, "%s: a tensor pointer is NULL", op);
    if (!aligned(a->key, 16) || !aligned(a->value, 16) || !aligned(a->key_rope, 16) || a->key_stride_t % 8 != 0 || a->key_stride_h % 8 != 0 ||
        a->value_stride_t % 8 != 0 || a->value_stride_h % 8 != 0 || a->key_rope_stride_t % 8 != 0 || a->key_rope_stride_h % 8 != 0)
        return fail(PTO_E_INVALID_ARG, "%s: keys and values must be 16-byte aligned, their strides multiples of 8 elements", op);
    if (!aligned(a->query, 2) || !aligned(a->query_rope, 2) || !aligned(a->out, 2) || !aligned(a->lse, 4) || !aligned(a->cu_seqlens_q, 4) ||
        !aligned(a->cu_seqlens_k, 4))
        return fail(PTO_E_INVALID_ARG, "%s: pointers must be aligned to their element size", op);
    constexpr int64_t most = (1ll << 32) / (2 * pto::PA_KEYS) - 256;
    if (a->key_stride_t < 0 || a->key_stride_t > most || a->value_stride_t < 0 || a->value_stride_t > most || a->key_rope_stride_t < 0 || a->key_rope_stride_t > most)
        return fail(PTO_E_INVALID_ARG, "%s: key and value token strides must be in [0, %lld]", op, (long long)most);
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "%s: no usable device is current", op);
    const PromptPlan pl = attention_plan(a, window, sinks);
    const size_t need = pl.o_bytes + pl.ml_bytes;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need))
        return fail(PTO_E_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", op, need, a->workspace ? a->workspace_bytes : (size_t)0);
    if (!aligned(a->workspace, 16)) return fail(PTO_E_INVALID_ARG, "%s: the workspace must be 16-byte aligned", op);
    if (pl.workgroups > 0x7ffffff0ll)
        return fail(PTO_E_INVALID_ARG, "%s: the call exceeds the largest launch", op);

    pto::PaParams p{};
    p.q = static_cast<const uint16_t *>(a->query);
    p.qr = static_cast<const uint16_t *>(a->query_rope);
    p.k = static_cast<const uint16_t *>(a->key);
    p.kr = static_cast<const uint16_t *>(a->key_rope);
    p.v = static_cast<const uint16_t *>(a->value);
    p.out = static_cast<uint16_t *>(a->out);
    p.lse = a->lse;
    p.part_o = static_cast<float *>(a->workspace);
    p.part_ml = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + pl.o_bytes);
    p.cu_q = a->cu_seqlens_q;
    p.cu_k = a->cu_seqlens_k;
    p.q_t = a->query_stride_t, p.q_h = a->query_stride_h;
    p.qr_t = a->query_rope_stride_t, p.qr_h = a->query_rope_stride_h;
    p.k_t = a->key_stride_t, p.k_h = a->key_stride_h;
    p.kr_t = a->key_rope_stride_t, p.kr_h = a->key_rope_stride_h;
    p.v_t = a->value_stride_t, p.v_h = a->value_stride_h;
    p.o_t = a->out_stride_t, p.o_h = a->out_stride_h;
    p.total_q = a->total_q, p.total_k = a->total_k;
    p.B = (int)a->b;
    p.kv_heads = (int)a->kv_heads;
    p.group = (int)(a->heads / a->kv_heads);
    p.d = (int)a->d;
    p.rope = a->query_rope != nullptr;
    p.fp16 = a->fp16 != 0;
    p.causal = a->causal != 0;
    p.q_whole = aligned(a->query, 16) && aligned(a->query_rope, 16) && a->query_stride_t % 8 == 0 && a->query_stride_h % 8 == 0 &&
                a->query_rope_stride_t % 8 == 0 && a->query_rope_stride_h % 8 == 0;
    p.window = (int)window;
    p.sinks = (int)sinks;
    p.most_tiles = pl.most_tiles;
    p.splits = pl.splits;
    p.split_tiles = pl.split_tiles;
    p.waves = pl.waves;
    p.grid = (int)pl.workgroups;
    p.cus = cu_count();
    p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
    const hipError_t e = pto::prompt_attention_launch(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "%s: launch failed: %s", op, hipGetErrorString(e));
    return PTO_OK;
}

int window_check(const PtoPromptWindowArgs *a)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "prompt_window_attention: args is NULL");
    if (a->window < 1 || a->window > MOST_TOKENS || a->sinks < 0 || a->sinks > MOST_TOKENS)
        return fail(PTO_E_INVALID_ARG, "prompt_window_attention: window must be in [1, 2^30], sinks in [0, 2^30]");
    if (!a->prompt.causal) return fail(PTO_E_INVALID_ARG, "prompt_window_attention: a window is causal");
    return attention_check("prompt_window_attention", &a->prompt);
}

}  // namespace

extern "C" {

int pto_rotary_tables_launch(const PtoRotaryTablesArgs *a, void *hip_stream)
{
    const int rc = tables_check(a);
    if (rc != PTO_OK || a->t == 0) return rc;
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "rotary_tables: no usable device is current");
    pto::RotaryTablesParams p;
    p.positions = a->positions;
    p.freq = a->frequencies;
    p.cos = a->cos;
    p.sin = a->sin;
    p.T = a->t;
    p.pairs = (int)a->pairs;
    p.wide = a->positions_int64 != 0;
    p.dtype = a->dtype;
    p.factor = (float)a->factor;
    const hipError_t e = pto::rotary_tables_launch(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "rotary_tables: launch failed: %s", hipGetErrorString(e));
    return PTO_OK;
}

int pto_rotary_launch(const PtoRotaryArgs *a, void *hip_stream)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "rotary: args is NULL");
    if (a->t < 0 || a->t > MOST_TOKENS) return fail(PTO_E_INVALID_ARG, "rotary: t out of range");
    if (a->pairs < 8 || a->pairs % 8 != 0 || a->pairs > pto::ROT_MAX_PAIRS)
        return fail(PTO_E_INVALID_ARG, "rotary: pairs must be a multiple of 8, up to %d (got %lld)", pto::ROT_MAX_PAIRS, (long long)a->pairs);
    if (!dtype_known(a->dtype)) return fail(PTO_E_INVALID_ARG, "rotary: unknown dtype code %d", a->dtype);
    if (a->layout < PTO_ROPE_HALF || a->layout > PTO_ROPE_DEINTERLEAVED) return fail(PTO_E_INVALID_ARG, "rotary: unknown layout %d", a->layout);
    if (!std::isfinite(a->factor)) return fail(PTO_E_INVALID_ARG, "rotary: factor is not finite");
    if (a->t == 0) return PTO_OK;
    if (!a->positions || !a->frequencies) return fail(PTO_E_INVALID_ARG, "rotary: a tensor pointer is NULL");
    if (!aligned(a->positions, a->positions_int64 ? 8 : 4) || !aligned(a->frequencies, 8))
        return fail(PTO_E_INVALID_ARG, "rotary: pointers must be aligned to their element size");
    pto::RotaryParams p{};
    int rc = rotary_side(a->query, "query", a->pairs, a->dtype, p.side[0]);
    if (rc != PTO_OK) return rc;
    if (a->key.in) {
        rc = rotary_side(a->key, "key", a->pairs, a->dtype, p.side[1]);
        if (rc != PTO_OK) return rc;
    }
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "rotary: no usable device is current");
    p.positions = a->positions;
    p.freq = a->frequencies;
    p.T = a->t;
    p.pairs = (int)a->pairs;
    p.wide = a->positions_int64 != 0;
    p.dtype = a->dtype;
    p.layout = a->layout;
    p.factor = (float)a->factor;
    p.cus = cu_count();
    const hipError_t e = pto::rotary_launch(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "rotary: launch failed: %s", hipGetErrorString(e));
    return PTO_OK;
}

int pto_cache_write_launch(const PtoCacheWriteArgs *a, void *hip_stream)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "cache_write: args is NULL");
    if (a->t < 0 || a->t > MOST_TOKENS) return fail(PTO_E_INVALID_ARG, "cache_write: t out of range");
    if (!dtype_known(a->dtype)) return fail(PTO_E_INVALID_ARG, "cache_write: unknown dtype code %d", a->dtype);
    pto::CacheWriteParams p{};
    const int rc = cache_of("cache_write", a->nope, a->rope_cache, a->scales, a->packed != 0, a->cache_rows, p.cache);
    if (rc != PTO_OK) return rc;
    if (a->t == 0) return PTO_OK;
    if (!a->latent || !a->rope || !a->cache_index) return fail(PTO_E_INVALID_ARG, "cache_write: a tensor pointer is NULL");
    if (!aligned(a->latent, element(a->dtype)) || !aligned(a->rope, element(a->dtype)) || !aligned(a->cache_index, 8) || !aligned(a->values, 2))
        return fail(PTO_E_INVALID_ARG, "cache_write: pointers must be aligned to their element size");
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "cache_write: no usable device is current");
    p.latent = a->latent;
    p.rope = a->rope;
    p.latent_t = a->latent_stride;
    p.rope_t = a->rope_stride;
    p.index = reinterpret_cast<const long long *>(a->cache_index);
    p.values = static_cast<uint16_t *>(a->values);
    p.values_t = a->values_stride;
    p.T = a->t;
    p.dtype = a->dtype;
    p.one_rounding = a->prolog_steps != 0;
    const hipError_t e = pto::cache_write_launch(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "cache_write: launch failed: %s", hipGetErrorString(e));
    return PTO_OK;
}

int pto_cache_read_launch(const PtoCacheReadArgs *a, void *hip_stream)
{
    if (!a) return fail(PTO_E_INVALID_ARG, "cache_read: args is NULL");
    if (a->rows < 0 || a->rows > MOST_TOKENS || a->b < 1 || a->b > (1ll << 24)) return fail(PTO_E_INVALID_ARG, "cache_read: b or rows out of range");
    if (a->block_size < 1 || a->block_size > (1ll << 30) || a->max_blocknum_perbatch < 1 || a->max_blocknum_perbatch > (1ll << 30))
        return fail(PTO_E_INVALID_ARG, "cache_read: block_size and max_blocknum_perbatch must be in [1, 2^30]");
    pto::CacheReadParams p{};
    const int rc = cache_of("cache_read", a->nope, a->rope_cache, a->scales, a->packed != 0, a->cache_rows, p.cache);
    if (rc != PTO_OK) return rc;
    if (a->rows == 0) return PTO_OK;
    if (!a->block_table || !a->cu_seqlens || !a->latent || !a->key_rope) return fail(PTO_E_INVALID_ARG, "cache_read: a tensor pointer is NULL");
    if (!aligned(a->block_table, 4) || !aligned(a->cu_seqlens, 4) || !aligned(a->first, 4) || !aligned(a->latent, 2) || !aligned(a->key_rope, 2))
        return fail(PTO_E_INVALID_ARG, "cache_read: pointers must be aligned to their element size");
    if (cu_count() <= 0) return fail(PTO_E_NO_DEVICE, "cache_read: no usable device is current");
    p.bt = a->block_table;
    p.cu = a->cu_seqlens;
    p.first = a->first;
    p.latent = static_cast<uint16_t *>(a->latent);
    p.rope = static_cast<uint16_t *>(a->key_rope);
    p.latent_t = a->latent_stride;
    p.rope_t = a->key_rope_stride;
    p.rows = a->rows;
    p.B = (int)a->b;
    p.maxblk = (int)a->max_blocknum_perbatch;
    p.bs = (int)a->block_size;
    const hipError_t e = pto::cache_read_launch(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return fail(PTO_E_LAUNCH, "cache_read: launch failed: %s", hipGetErrorString(e));
    return PTO_OK;
}

int pto_prompt_attention_workspace_bytes(const PtoPromptAttentionArgs *a, size_t *bytes)
{
    if (!bytes) return fail(PTO_E_INVALID_ARG, "prompt_attention: bytes is NULL");
    const int rc = attention_check("prompt_attention", a);
    if (rc != PTO_OK) return rc;
    const PromptPlan pl = attention_plan(a, 0, 0);
    *bytes = pl.o_bytes + pl.ml_bytes;
    return PTO_OK;
}

int pto_prompt_attention_plan(const PtoPromptAttentionArgs *a, PtoPromptPlan *plan)
{
    if (!plan) return fail(PTO_E_INVALID_ARG, "prompt_attention: plan is NULL");
    const int rc = attention_check("prompt_attention", a);
    if (rc != PTO_OK) return rc;
    const PromptPlan pl = attention_plan(a, 0, 0);
    plan->rows_per_workgroup = pl.waves * pto::PA_WAVE_ROWS;
    plan->key_splits = pl.splits;
    plan->split_keys = (int64_t)pl.split_tiles * pto::PA_KEYS;
    plan->workgroups = pl.workgroups;
    return PTO_OK;
}

int pto_prompt_attention_launch(const PtoPromptAttentionArgs *a, void *hip_stream)
{
    const int rc = attention_check("prompt_attention", a);
    return rc != PTO_OK ? rc : attention_launch("prompt_attention", a, 0, 0, hip_stream);
}

int pto_prompt_window_workspace_bytes(const PtoPromptWindowArgs *a, size_t *bytes)
{
    if (!bytes) return fail(PTO_E_INVALID_ARG, "prompt_window_attention: bytes is NULL");
    const int rc = window_check(a);
    if (rc != PTO_OK) return rc;
    const PromptPlan pl = attention_plan(&a->prompt, a->window, a->sinks);
    *bytes = pl.o_bytes + pl.ml_bytes;
    return PTO_OK;
}

int pto_prompt_window_launch(const PtoPromptWindowArgs *a, void *hip_stream)
{
    const int rc = window_check(a);
    return rc != PTO_OK ? rc : attention_launch("prompt_window_attention", &a->prompt, a->window, a->sinks, hip_stream);
}

}  // extern "C"
