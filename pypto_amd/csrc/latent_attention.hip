// Attention over the cached latents of whole sequences, gfx950: every key, the last ones of a window and a few first ones, or the context and a
// tree of drafted tokens.  The absorbed form: a key row is 512 int8 with four scales and 64 bf16 rope channels, values are its 512, all
// heads share them.
//
// Row r of a sequence is (token r / heads, head r % heads); a workgroup takes 64 consecutive rows, whichever tokens they are of, so that heads and
// tokens alike share the keys that are read.  Tiles of 32 keys, eight waves:
//   scores: wave (kh, hq) multiplies the 16 keys of half kh with rows 16*hq .. +15 over all 576 channels
//           (v_mfma_f32_16x16x32_bf16: the accumulator's lane (row, quarter) holds four keys of one row), nothing to add up;
//   softmax: of those four scores, in place; the probabilities go round through LDS as the B operand of the second product;
//   values: wave w owns 64 value channels of all 64 rows; each transposed V operand serves two products.
// The products against V of tile n - 1 run beside the scores and the softmax of tile n: one barrier per tile, three tile buffers.
// Cache rows travel to registers two tiles ahead of their use, their pages one more, and are de-quantised on the way into LDS.
//
// Division of the work.  A row tile takes as many units as it has key tiles and LA_OPEN more for its beginning and end; all units lie in one line,
// which the workgroups divide evenly, an XCD's neighbouring pieces to neighbouring workgroups.  A boundary near a row tile's edge moves there.
// Where one falls inside, both sides write their sums, maxima and 512 sums of products, in fp32, and a second launch joins them: two pieces at most
// to a workgroup, so the memory for them does not depend on lengths, which the host does not know.
#include <type_traits>

#include "common.h"
#include "serving_ops.h"

namespace pto {
namespace {

constexpr int DN = 512, DR = 64;
constexpr int KT = LA_KEYS;
constexpr int PITCH = (DN + DR + 8) * 2;                  // bytes of a tile row: 512 latent and 64 rope channels as bf16, 16 spare
constexpr int TILE = KT * PITCH;
constexpr int P_AT = 3 * TILE;                            // two buffers of P^T: [row half][k-step][lane] 16 bytes
constexpr int P_BYTES = 4096;
constexpr int MAX_AT = P_AT + 2 * P_BYTES;                // [key half][64 rows] fp32: maxima (and at the end the sums)
constexpr int ALPHA_AT = MAX_AT + 2 * 64 * 4;             // [64 rows] fp32: rescale factors (at the end 1 / sum)
constexpr int FLAG_AT = ALPHA_AT + 64 * 4;                // two words: the last tile whose maxima moved, by parity of the tile
constexpr int POOL = FLAG_AT + 16;
constexpr int Q_ROPE_AT = LA_ROWS * DN * 2;               // query staging: 64 rows x 1024 bytes, then 64 x 128
constexpr float TAU = 8.0f;                               // log2 units: the reference maximum moves only when exceeded by 2^8
constexpr float LOW = -1.7e38f;                           // reference maximum of a row that has seen no key yet
constexpr int PIECE = LA_ROWS * DN;                       // floats of a piece's sums

__device__ const u32x4 no_page[4 * (DN + 2 * DR + 16) / 16] = {};      // what four keys without a page read, a whole row of the cache each

// Row i of a tile's score operand (and of the score accumulator) is key tile_row_of(i) of the tile: the two middle bits of i move below its two
// lowest.  A transposing V^T read then addresses keys r, r+4, r+8, r+12 with each of its half-waves, four rows whose 64-byte pieces lie
// 16 banks apart at this pitch; any 16 consecutive keys, in whatever order, still serve the score operand reads without a conflict.
__device__ __forceinline__ constexpr int tile_row_of(const int i) { return (i & 16) | ((i & 3) << 2) | ((i >> 2) & 3); }

__device__ __forceinline__ void both_halves(const float x, float &lo, float &hi)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    lo = __uint_as_float(r[0]);
    hi = __uint_as_float(r[1]);
}
// max and sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48, in every one of them
__device__ __forceinline__ float quarters_max(const float x)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    float lo, hi;
    both_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])), lo, hi);
    return fmaxf(lo, hi);
}
__device__ __forceinline__ float quarters_sum(const float x)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    float lo, hi;
    both_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]), lo, hi);
    return lo + hi;
}

// one dword of int8 times the scale: two dwords of bf16, each product rounded to fp32 and then to bf16
__device__ __forceinline__ u32x2 dequant_dword(const uint32_t r, const float sc)
{
    float f0, f1, f2, f3;
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f0) : "v"(r));
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f1) : "v"(r));
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f2) : "v"(r));
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f3) : "v"(r));
    return u32x2{pack_bf16x2(f0 * sc, f1 * sc), pack_bf16x2(f2 * sc, f3 * sc)};
}

// (what hangs on the lane alone is made anew for each row tile instead of being kept)
__device__ __forceinline__ uint32_t opaque(uint32_t x)
{
    asm("" : "+v"(x));
    return x;
}
template <typename T>
__device__ __forceinline__ T global(const uint8_t *base, const uint32_t offset)
{
    return *(const __attribute__((address_space(1))) T *)((const __attribute__((address_space(1))) uint8_t *)base + offset);
}
// a scalar load, of what no launch that this one may run beside writes
template <typename T>
__device__ __forceinline__ T constant(const T *at)
{
    return *(const __attribute__((address_space(4))) T *)at;
}
// sums of x over this lane and all lanes before it
__device__ __forceinline__ long long wave_sums(long long x)
{
    auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)((uint64_t)x >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
        x += (long long)((uint64_t)lo | ((uint64_t)hi << 32));
    };
    const std::integral_constant<int, 0xf> all;
    add(std::integral_constant<int, 0x111>{}, all);        // row_shr:1, 2, 4, 8: within rows of sixteen lanes
    add(std::integral_constant<int, 0x112>{}, all);
    add(std::integral_constant<int, 0x114>{}, all);
    add(std::integral_constant<int, 0x118>{}, all);
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});     // row_bcast:15: rows 0 and 2 into 1 and 3
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});     // row_bcast:31: the lower half into the upper
    return x;
}
__device__ __forceinline__ long long first_of(const long long x)
{
    return (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32));
}

// A sequence as the kernel takes it: whatever the tables say, inside the tensors.
struct Sequence {
    int q0, n, keys;                                       // first token, tokens, keys
    int tiles, row_tiles;                                  // units of a row tile but LA_OPEN; row tiles
};
__device__ __forceinline__ void count_tiles(const LaParams &p, Sequence &c)
{
    c.row_tiles = (c.n * p.heads + LA_ROWS - 1) / LA_ROWS;
    c.tiles = (c.keys + KT - 1) / KT;
    c.tiles = c.tiles < p.most_tiles ? c.tiles : p.most_tiles;
}
__device__ __forceinline__ Sequence sequence(const LaParams &p, const int b)
{
    Sequence c;
    const int total = (int)p.total_q;
    int lo = p.cu_q[b], hi = p.cu_q[b + 1], keys = p.lens[b];
    lo = lo < 0 ? 0 : (lo > total ? total : lo);
    hi = hi < lo ? lo : (hi > total ? total : hi);
    keys = keys < 0 ? 0 : (keys > p.most_keys ? p.most_keys : keys);
    c.q0 = lo, c.n = hi - lo, c.keys = keys;
    count_tiles(p, c);
    return c;
}

// x / d for 0 <= x < 2^51, d >= 1 and a quotient below 2^31: of the product with 1 / d the whole part is off by one at most
__device__ __forceinline__ int quotient(const long long x, const int d)
{
    int q = (int)((double)x * (1.0 / (double)d));
    if ((long long)q * d > x) --q;
    if ((long long)(q + 1) * d <= x) ++q;
    return q;
}

// The row tile that a unit is in.
struct Place {
    int b, q0, n, keys, tiles, row_tile, ordinal;          // ordinal: among the row tiles of all sequences
    long long begin;                                       // its first unit
};

// A boundary `x` units into a row tile of `len`, moved to its edge where that is near.
constexpr int NEAR_BEGIN = LA_OPEN + 3, NEAR_END = 3;
__device__ __forceinline__ int moved(const int x, const int len) { return x <= NEAR_BEGIN ? 0 : (x >= len - NEAR_END ? len : x); }

constexpr int THREADS = LA_THREADS;

// QUADS: pages and the cache hold whole fours of rows.
template <bool QUADS>
__global__ __launch_bounds__(THREADS) void latent_attention_kernel(const LaParams p)
{
    __shared__ __attribute__((aligned(16))) uint8_t pool[POOL];

    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hq = w & 3;                                  // scores: rows 16*hq .. +15 of the workgroup's 64,
    const int kh = w >> 2;                                 // the half kh of the tile's keys
    const uint32_t pool_lds = (uint32_t)(uintptr_t)(lds_byte_t *)pool;

    // Units and row tiles of the sequences up to each: an entry to a thread, of as many sequences as that takes.
    __shared__ long long upto[THREADS], of_waves[THREADS / 64];
    __shared__ int tiles_upto[THREADS], tiles_of_waves[THREADS / 64];
    __shared__ int seq_q0[THREADS], seq_n[THREADS], seq_keys[THREADS];         // of an entry's first sequence
    const int per_entry = p.per_entry, entries = p.seq_entries;
    {
        long long mine = 0;
        int row_tiles = 0;
        for (int j = 0; j < per_entry; ++j) {
            const int b = tid * per_entry + j;
            if (b < p.B) {
                const Sequence c = sequence(p, b);
                if (j == 0) seq_q0[tid] = c.q0, seq_n[tid] = c.n, seq_keys[tid] = c.keys;
                mine += (long long)c.row_tiles * (c.tiles + LA_OPEN), row_tiles += c.row_tiles;
            }
        }
        mine = wave_sums(mine);
        const long long both = wave_sums((long long)row_tiles);
        if ((tid & 63) == 63) of_waves[w] = mine, tiles_of_waves[w] = (int)both;
        __syncthreads();
        int before = 0;
        for (int i = 0; i < w; ++i) mine += of_waves[i], before += tiles_of_waves[i];
        upto[tid] = mine;
        tiles_upto[tid] = (int)both + before;
        __syncthreads();
    }
    const long long units = first_of(upto[THREADS - 1]);
    const int row_tiles = __builtin_amdgcn_readfirstlane(tiles_upto[THREADS - 1]);
    auto place_of = [&](const long long u) __attribute__((always_inline)) {
        int e = 0;                                         // entries that end in front of u
        for (int i = 0; i < entries; i += 64) e += __popcll(__ballot(upto[i + (tid & 63)] <= u));
        long long first = e > 0 ? first_of(upto[e - 1]) : 0;
        int tiles_before = e > 0 ? __builtin_amdgcn_readfirstlane(tiles_upto[e - 1]) : 0;
        Place at;
        at.b = e * per_entry;
        Sequence c;
        c.q0 = __builtin_amdgcn_readfirstlane(seq_q0[e]), c.n = __builtin_amdgcn_readfirstlane(seq_n[e]), c.keys = __builtin_amdgcn_readfirstlane(seq_keys[e]);
        count_tiles(p, c);
        for (int j = 1; j < per_entry; ++j) {              // (only of more than THREADS sequences)
            const long long next = first + (long long)c.row_tiles * (c.tiles + LA_OPEN);
            if (next > u || at.b + 1 >= p.B) break;
            first = next, tiles_before += c.row_tiles, ++at.b;
            c = sequence(p, at.b);
        }
        at.q0 = c.q0, at.n = c.n, at.keys = c.keys, at.tiles = c.tiles;
        at.row_tile = __builtin_amdgcn_readfirstlane(quotient(u - first, c.tiles + LA_OPEN));
        at.ordinal = tiles_before + at.row_tile;
        at.begin = first + (long long)at.row_tile * (c.tiles + LA_OPEN);
        return at;
    };
    // workgroups that take part, so that none gets less than LA_LEAST units; this one's number among them
    const long long most = (long long)p.groups * LA_LEAST;
    const int pieces = units < most ? (int)units / LA_LEAST : p.groups, groups = pieces > 0 ? pieces : 1;
    const int per_xcd = (groups + 7) / 8, slot = blockIdx.x >> 3;
    const int g = (int)(blockIdx.x & 7) * per_xcd + slot;
    const bool there = slot < per_xcd && g < groups;
    // Which row tiles are joined, and from how many pieces: said by the workgroup that has the first of them, for every other entry that there are none.
    if (tid == 0) {
        if (p.by_tile) {
            for (int i = row_tiles + (int)blockIdx.x; i < p.entries; i += (int)gridDim.x) p.joins[4 * i + 1] = 0;
        } else if (!there) {
            p.joins[4 * blockIdx.x + 1] = 0;
        }
    }
    if (!there) return;
    // the line's even divisions: units * i / groups
    long long share = (long long)((double)units / (double)groups);
    if (share * groups > units) --share;
    const int rest = (int)(units - share * groups);
    auto division = [&](const int i) { return share * i + (rest * i) / groups; };
    long long u = 0, u_end = units, want = division(g + 1 < groups ? g + 1 : g);
    int step = g + 1 < groups ? 0 : 1;                     // looked for: this workgroup's end, its beginning, the next row tile
    bool said = false;                                     // (not by_tile) this workgroup's entry is written
    bool first_segment = true;

    while (units > 0) {
        const int l = (int)opaque(tid & 63), half = l >> 5, col = l & 31, l16 = l & 15, quarter = l >> 4;
        const Place at = place_of(want);
        if (step < 2) {
            const long long edge = at.begin + moved((int)(want - at.begin), at.tiles + LA_OPEN);
            if (step == 0) {
                u_end = edge, want = division(g), step = 1;
                continue;
            }
            u = edge, step = 2;
            if (u >= u_end) break;
            if (u == at.begin + at.tiles + LA_OPEN) {
                want = u;
                continue;
            }
        }
        const int len = at.tiles + LA_OPEN;
        const long long end = at.begin + len;
        const long long to = u_end < end ? u_end : end;
        const bool whole = u == at.begin && to == end;
        int i_begin = (int)(u - at.begin) - LA_OPEN;
        i_begin = i_begin < 0 ? 0 : i_begin;
        int i_end = (int)(to - at.begin) - LA_OPEN;

        // the piece's place, and what is to be joined
        const int piece = 2 * g + (first_segment ? 0 : 1);
        const int rows = at.n * p.heads, row0 = at.row_tile * LA_ROWS;
        if (tid == 0 && u == at.begin && (p.by_tile || !whole)) {
            int n = 0;
            if (!whole) {                                  // pieces: one more than there are boundaries inside, those before unit end - NEAR_END
                const long long edge = end - NEAR_END;
                n = (int)((double)edge * (double)groups / (double)units) - g;
                n = n > 1 ? n - 1 : 1;
                while (g + n < groups && division(g + n) < edge) ++n;
            }
            int32_t *const join = p.joins + 4 * (p.by_tile ? at.ordinal : (int)blockIdx.x);
            join[0] = piece, join[1] = n, join[2] = at.q0 * p.heads + row0, join[3] = rows - row0 < LA_ROWS ? rows - row0 : LA_ROWS;
            said = true;
        }

        // What the row tile's tokens see, and which of the units are which tiles of keys.
        const int last = rows - 1 - row0 < LA_ROWS - 1 ? rows - 1 - row0 : LA_ROWS - 1;       // its last row
        const int tok0 = divide(row0, p.of_heads), tok1 = divide(row0 + last, p.of_heads);
        const bool tree = p.mask != nullptr;
        const int context = at.keys - at.n > 0 ? at.keys - at.n : 0;                           // keys before the tree
        auto sees_of = [&](const int tok) {
            const int s = tok + 1 + at.keys - at.n;
            return tree ? at.keys : (s < 0 ? 0 : s);
        };
        auto from_of = [&](const int sees) { return p.window > 0 && sees > p.window ? sees - p.window : 0; };
        const int least = tree ? context : sees_of(tok0), most = sees_of(tok1);                // keys that all, that some rows see (but for windows)
        const int low_first = from_of(sees_of(tok0)), low_last = from_of(sees_of(tok1));       // where windows begin
        const int key_tiles = (most + KT - 1) / KT;
        int sink_tiles = (p.sinks + KT - 1) / KT;
        sink_tiles = sink_tiles < low_first / KT ? sink_tiles : low_first / KT;
        const int skip = low_first / KT - sink_tiles;
        i_end = i_end < key_tiles - skip ? i_end : key_tiles - skip;
        const int ntiles = i_end > i_begin ? i_end - i_begin : 0;
        auto key_of_tile = [&](const int n) {              // the first key of tile n of this piece
            const int i = i_begin + (n < ntiles ? n : ntiles - 1);
            return KT * (i < sink_tiles ? i : i + skip);
        };
        // of this lane's row of scores
        const int my_row = row0 + 16 * hq + l16;
        const int my_tok = divide(my_row < rows ? my_row : rows - 1, p.of_heads);
        const int my_sees = sees_of(my_tok), my_from = from_of(my_sees);
        const unsigned long long *const my_mask = tree ? p.mask + (long long)(at.q0 + my_tok) * p.words : nullptr;

        f32x16 o[4];                                       // block 2*hb + d: rows 32*hb .., value channels 64w + 32d ..
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
        float m_run = LOW;                                 // of row 16*hq + l16: reference maximum, log2 domain,
        float l_run = 0.f;                                 // and this lane's share of the sum of exp2(s - m_run)

        if (ntiles > 0) {                                  // uniform
            // The queries, staged through LDS in the tile buffers 0 and 1: wave w asks for rows 8w .. 8w+7, a row's latent part per request,
            // 16-byte chunk i of row j at i ^ (j & 15) so that the fragment reads touch every bank once.  Rows past the last one read it
            // and are never stored.
            static_assert(Q_ROPE_AT + LA_ROWS * DR * 2 <= 2 * TILE, "the first tile goes to buffer 2");
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 8 * w + i, r = row0 + (j < last ? j : last);
                const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                dma16_base(p.q + (long long)(at.q0 + tok) * p.q_t + (long long)head * p.q_h, (uint32_t)(16 * (l ^ (j & 15))), pool_lds + j * (DN * 2));
            }
            {
                const int j = 8 * w + (l >> 3), r = row0 + (j < last ? j : last);
                const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                dma16(p.qr + (long long)(at.q0 + tok) * p.qr_t + (long long)head * p.qr_h + 8 * ((l & 7) ^ (l >> 3)), pool_lds + Q_ROPE_AT + w * 1024);
            }

            // Gather: wave w takes keys 4w .. 4w+3 of every tile, a quarter of its lanes each, a lane 32 channels of the latents (one scale) and
            // four of the rope part.  QUADS: the four are neighbours in the cache, so one scalar look-up and one address serve them.  Keys past
            // the sequence's last one are those of the same four that are left in its page (their scores are hidden, and check_scales
            // keeps what they hold out of the sums), else stand in with the last one.
            struct Raw {
                u32x4 v[2];
                float sc;
                u32x2 rope;
            };
            Raw raw[2];                                    // tile n in raw[n & 1]
            struct Page {
                int page, within;
            };
            auto page_of = [&](const int n) __attribute__((always_inline)) {
                int key = key_of_tile(n) + 4 * w + (QUADS ? 0 : quarter);
                const int last_key = QUADS ? (at.keys - 1) & ~3 : at.keys - 1;
                key = key < last_key ? key : last_key;
                const int block = divide(key, p.of_bs);    // (the block table has it: at.keys is no more than its pages hold)
                const int32_t *const entry = p.bt + (long long)at.b * p.maxblk + block;
                return Page{QUADS ? constant<int32_t>(entry) : *entry, key - block * p.bs};
            };
            const uint32_t rows_on = QUADS ? quarter : 0;
            const uint32_t v_off = rows_on * (uint32_t)p.cache.nope_pitch + 32 * l16, sc_off = rows_on * (uint32_t)p.cache.scale_pitch + 4 * (l16 >> 2),
                           rope_off = rows_on * (uint32_t)p.cache.rope_pitch + 8 * l16;
            auto gather = [&](Raw &r, const Page k) __attribute__((always_inline)) {
                const long long row = (long long)k.page * p.bs + k.within;
                const bool there = k.page >= 0 && row < p.cache.rows;
                const uint8_t *const none = reinterpret_cast<const uint8_t *>(no_page);
                const uint8_t *const v = there ? p.cache.nope + row * p.cache.nope_pitch : none;
                const uint8_t *const sc = there ? p.cache.scale + row * p.cache.scale_pitch : none;
                const uint8_t *const rope = there ? p.cache.rope + row * p.cache.rope_pitch : none;
                r.v[0] = global<u32x4>(v, v_off);
                r.v[1] = global<u32x4>(v + 16, v_off);
                r.sc = global<float>(sc, sc_off);
                r.rope = global<u32x2>(rope, rope_off);
            };
            // A scale that is no number, or with which 127 steps are not finite, would be in the sums of rows that do not see the key (0 times it):
            // such a group's values become zeros and the key's rope channels, which are in scores alone, no numbers.  A row that sees the
            // key is then no number, others are not touched.
            auto check_scales = [&](Raw &r) __attribute__((always_inline)) {
                const bool bad = !(fabsf(r.sc) < 2.6e36f);
                const uint64_t any = __ballot(bad);
                if (__builtin_expect(any != 0, 0)) {
                    r.sc = bad ? 0.f : r.sc;
                    if (((any >> (16 * quarter)) & 0xffff) != 0) r.rope = u32x2{0x7fc07fc0u, 0x7fc07fc0u};
                }
            };
            // The tile's rows into LDS, in eight pieces of a dword per lane and one of the rope channels.  Of a row's 64 latent pieces of eight
            // channels number 4 j + k lies at k * 16 + j: a lane's four pieces are one of each k, and lanes next to each other write next to
            // each other.
            const uint32_t emit_off = (uint32_t)((4 * w + quarter) * PITCH + 16 * l16);
            const uint32_t emit_rope_off = (uint32_t)((4 * w + quarter) * PITCH + DN * 2 + 8 * l16);
            u32x4 dq;
            auto emit = [&](Raw &r, const uint32_t tile, const int d) __attribute__((always_inline)) {
                if (d == 0) check_scales(r);
                if (d == 8) {
                    *reinterpret_cast<u32x2 *>(pool + tile + emit_rope_off) = r.rope;
                } else {
                    const u32x2 x = dequant_dword(r.v[d >> 2][d & 3], r.sc);
                    if (d & 1) {
                        dq[2] = x[0], dq[3] = x[1];
                        *reinterpret_cast<u32x4 *>(pool + tile + emit_off + 256 * (d >> 1)) = dq;
                    } else {
                        dq[0] = x[0], dq[1] = x[1];
                    }
                }
            };
            Page page = page_of(0), page1 = page_of(1), page2 = page_of(2), page3 = page_of(3);
            gather(raw[0], page);
            gather(raw[1], page1);
            // the waves' own queries have landed; those of the others when every wave has come here
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            __syncthreads();
            // Q^T: of the latent part lane (row, quarter) holds the channels of the tile rows' 16-byte pieces at 16*quarter + ks, of
            // the rope part channels 16*quarter + 8*ks .. +7
            bf16x8 qf[18];
#pragma unroll
            for (int ks = 0; ks < 16; ++ks)
                qf[ks] = *reinterpret_cast<const bf16x8 *>(pool + (16 * hq + l16) * (DN * 2) + 16 * ((4 * ks + quarter) ^ l16));
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
                qf[16 + ks] = *reinterpret_cast<const bf16x8 *>(pool + Q_ROPE_AT + (16 * hq + l16) * (DR * 2) + 16 * ((2 * quarter + ks) ^ (l16 & 7)));
            // Scores are scaled inside the exponent (one multiply-add per key).  That wants a positive scale: the sign of a negative
            // one moves into Q^T (exact), and a zero one becomes the smallest normal number, under which every score up to 1e31 still
            // scales to an exponent that rounds to the same probabilities.
            float sc_log2 = p.scale_log2;
            if (sc_log2 < 0.f) {
                sc_log2 = -sc_log2;
#pragma unroll
                for (int i = 0; i < 18; ++i) qf[i] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, qf[i]) ^ 0x80008000u);
            }
            if (sc_log2 == 0.f) sc_log2 = 1.17549435e-38f;
            if (tid < 2) reinterpret_cast<int *>(pool + FLAG_AT)[tid] = -1;
#pragma unroll
            for (int d = 0; d < 9; ++d) emit(raw[0], 2 * TILE, d);
            gather(raw[0], page2);
            page2 = page_of(4);
            __syncthreads();

            // Score operand: row `a` of the wave's sixteen is key tile_row_of(16*kh + a); the accumulator then holds in lane
            // (row, quarter) the keys 4*quarter + r, the k-order of the second product's B operand.
            // (quarters 256 bytes apart: whichever sixteen lanes the LDS serves together, their rows alone decide the banks)
            const uint32_t kbase = (uint32_t)(tile_row_of(16 * kh + l16) * PITCH + 256 * quarter);
            const uint32_t krope = (uint32_t)(tile_row_of(16 * kh + l16) * PITCH + DN * 2 + 32 * quarter);
            const uint32_t vbase = (uint32_t)((half + 4 * (l16 >> 2)) * PITCH + 32 * ((l >> 4) & 1) + 8 * (l & 3) + 128 * w);
            const uint32_t pwrite = (uint32_t)(P_AT + (((hq >> 1) * 2 + kh) * 64 + 32 * (quarter & 1) + 16 * (hq & 1) + l16) * 16 + 8 * (quarter >> 1));
            int key_of[4];                                 // key of this lane's scores within the tile
#pragma unroll
            for (int e = 0; e < 4; ++e) key_of[e] = tile_row_of(16 * kh + 4 * quarter + e);

            bf16x8 vf[2][2], pf[2][2];
            f32x4 s;                                       // scores of the tile being multiplied
            float sv[4], mx = 0.f;                         // of the tile before it, and their maximum over the wave's keys
            float l_add = 0.f;                             // that tile's probabilities, not yet in l_run
            auto load_v = [&](const uint32_t tile, const int kk, const int d) __attribute__((always_inline)) {
                const uint16_t *a0 = reinterpret_cast<const uint16_t *>(pool + tile + vbase + (16 * kk) * PITCH + 64 * d);
                const s16x4 lo = lds_read_tr16(a0), hi = lds_read_tr16(a0 + PITCH);            // (two rows on)
                vf[kk][d] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            auto load_p = [&](const int pbuf, const int kk, const int hb) __attribute__((always_inline)) {
                pf[kk][hb] = *reinterpret_cast<const bf16x8 *>(pool + P_AT + pbuf * P_BYTES + ((hb * 2 + kk) * 64 + l) * 16);
            };
            auto first_vp = [&](const uint32_t tile, const int pbuf) __attribute__((always_inline)) {
                load_v(tile, 0, 0), load_v(tile, 0, 1);
                load_p(pbuf, 0, 0), load_p(pbuf, 0, 1);
            };
            // Scores of the tile in buffer `cur`, whose first AHEAD operands are in fa (or on their way).
            constexpr int AHEAD = 6;
            bf16x8 fa[18];
            auto read_k = [&](const uint32_t cur, const int m) __attribute__((always_inline)) {
                fa[m] = *reinterpret_cast<const bf16x8 *>(pool + cur + (m < 16 ? kbase + 16 * m : krope + 16 * (m - 16)));
            };
            auto first_k = [&](const uint32_t cur) __attribute__((always_inline)) {
#pragma unroll
                for (int m = 0; m < AHEAD; ++m) read_k(cur, m);
            };
            auto scores = [&](const uint32_t cur) __attribute__((always_inline)) {
                const f32x4 z = {};
                s = z;
#pragma unroll
                for (int m = 0; m < 18; ++m) {
                    s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[m], qf[m], s, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (m + AHEAD < 18) read_k(cur, m + AHEAD);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // The softmax of tile n.  The reference maximum follows the true one lazily: probabilities may reach 2^TAU, which fp32 sums and bf16 P
            // hold without loss.  A wave sees half of its rows' keys only; where one of its scores passes that bound it raises the
            // flag, and all waves take the tile's probabilities again (move_maxima) once the barrier has made the flag seen.
            auto probabilities = [&](const int pbuf) __attribute__((always_inline)) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i], sc_log2, -m_run));
                const u32x2 pk = {pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3])};
                *reinterpret_cast<u32x2 *>(pool + pwrite + pbuf * P_BYTES) = pk;
                l_add = (e[0] + e[1]) + (e[2] + e[3]);
            };
            auto take_scores = [&](const int n) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sv[e] = s[e];
                const int first = key_of_tile(n);
                const bool below = first + KT <= least;                                        // (uniform)
                if (!(below && (first >= low_last || first + KT <= p.sinks))) {
                    uint32_t drafted = ~0u;                // of the tile's keys, those in front of the tree and those of it that the row sees
                    if (tree && !below) {
                        const int node = first - context, at_word = node >> 6, shift = node & 63;
                        auto word = [&](const int i) { return i < 0 ? ~0ull : (i < p.words ? my_mask[i] : 0ull); };
                        const unsigned long long lo = word(at_word), hi = word(at_word + 1);
                        drafted = (uint32_t)((lo >> shift) | (shift ? hi << (64 - shift) : 0ull));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = first + key_of[e];
                        const bool seen = (key < my_sees) & ((key >= my_from) | (key < p.sinks)) & (((drafted >> key_of[e]) & 1) != 0);
                        sv[e] = seen ? sv[e] : -INFINITY;          // (without a branch for each score)
                    }
                }
                mx = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
            };
            auto softmax = [&](const int n, const int pbuf) __attribute__((always_inline)) {
                take_scores(n);
                probabilities(pbuf);
                if (__any(mx * sc_log2 > m_run + TAU)) reinterpret_cast<int *>(pool + FLAG_AT)[pbuf] = n;
            };
            // Probabilities of the tile whose scores are in sv, with the maxima moved where they passed the bound (always, on the
            // first tile): two barriers, every wave takes part.
            auto move_maxima = [&](const int pbuf, const bool first) __attribute__((always_inline)) {
                mx = quarters_max(mx);
                if (l < 16) reinterpret_cast<float *>(pool + MAX_AT)[64 * kh + 16 * hq + l16] = mx;
                __syncthreads();
                mx = fmaxf(mx, reinterpret_cast<const float *>(pool + MAX_AT)[64 * (kh ^ 1) + 16 * hq + l16]) * sc_log2;
                const bool upd = mx > m_run + TAU;
                const float m_new = upd ? mx : m_run;
                const float alpha = upd ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
                m_run = m_new;
                l_run *= alpha;
                if (kh == 0 && l < 16) reinterpret_cast<float *>(pool + ALPHA_AT)[16 * hq + l16] = alpha;
                probabilities(pbuf);
                __syncthreads();
                if (!first) {
#pragma unroll
                    for (int hb = 0; hb < 2; ++hb) {
                        const float a = reinterpret_cast<const float *>(pool + ALPHA_AT)[32 * hb + col];
#pragma unroll
                        for (int d = 0; d < 2; ++d)
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[2 * hb + d][e] *= a;
                    }
                }
            };
            // O^T += V^T . P^T of the tile in buffer `prev`, P^T in buffer pbuf, whose first operands are read; NEXT: beside them the
            // tile of r goes into buffer `next`, the rows of the tile two further are asked for, and the pages of the one behind it
            auto values = [&](auto next_tag, const int n4, const uint32_t prev, const uint32_t next, Raw &r, const int pbuf) __attribute__((always_inline)) {
                constexpr bool NEXT = decltype(next_tag)::value;
                Page further;
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int mp = 0; mp < 8; ++mp) {
                    const int kk = mp >> 2, d = (mp >> 1) & 1, hb = mp & 1;
                    o[2 * hb + d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[kk][d], pf[kk][hb], o[2 * hb + d], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (mp == 0) load_v(prev, 1, 0), load_p(pbuf, 1, 0);
                    if (mp == 1) load_v(prev, 1, 1), load_p(pbuf, 1, 1);
                    if (NEXT) {                            // (pages before rows: loads come back in order)
                        emit(r, next, mp);
                        if (mp == 4) further = page_of(n4);
                        if (mp == 7) emit(r, next, 8), gather(r, page), page = further;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // Every wave takes part in the tile's two halves of work in one of two orders: the waves of the keys' first half take the
            // scores of tile n first and then the products against V of tile n - 1, the others (the second wave of each SIMD) the
            // products first, so that one's LDS reads and vector work stand beside the other's products.
            auto moved_word = [&](const int pbuf) { return reinterpret_cast<const int *>(pool + FLAG_AT)[pbuf]; };
            uint32_t cur = 2 * TILE, next = 0, prev = TILE;                                    // buffers of tiles n, n + 1, n - 1
            auto turn = [&](auto parity, const int n) __attribute__((always_inline)) {
                constexpr int PAR = decltype(parity)::value;                                   // n & 1
                constexpr int pbuf = PAR ^ 1;                                                  // of tile n - 1
                if (kh == 0) {
                    first_k(cur);
                    scores(cur);
                }
                const int moved_at = moved_word(pbuf);
                first_vp(prev, pbuf);
                if (__builtin_expect(__builtin_amdgcn_readfirstlane(moved_at) == n - 1, 0)) {  // rare
                    move_maxima(pbuf, false);
                    first_vp(prev, pbuf);
                }
                l_run += l_add;
                if (kh == 0) softmax(n, PAR);
                values(std::true_type{}, n + 4, prev, next, raw[PAR ^ 1], pbuf);
                if (kh == 1) {
                    first_k(cur);
                    scores(cur);
                    softmax(n, PAR);
                }
                __syncthreads();
                const uint32_t third = prev;
                prev = cur;
                cur = next;
                next = third;
            };
            // the first tile: its maxima are moved at once
            first_k(cur);
            scores(cur);
#pragma unroll
            for (int d = 0; d < 9; ++d) emit(raw[1], next, d);
            gather(raw[1], page3);
            page = page2;                                  // of tile n + 3
            take_scores(0);
            move_maxima(0, true);
            prev = cur;
            cur = next;
            next = TILE;
            int n = 1;
            for (; n + 1 < ntiles; n += 2) {               // (two to a trip without a way out between them: exits inside make
                turn(std::integral_constant<int, 1>{}, n); // the compiler wait for every request)
                turn(std::integral_constant<int, 0>{}, n + 1);
            }
            if (n < ntiles) turn(std::integral_constant<int, 1>{}, n);
            // the products against V of the last tile
            const int pbuf = (ntiles & 1) ^ 1;
            if (__builtin_amdgcn_readfirstlane(moved_word(pbuf)) == ntiles - 1) move_maxima(pbuf, false);
            l_run += l_add;
            first_vp(prev, pbuf);
            values(std::false_type{}, 0, prev, 0, raw[0], pbuf);
        }

        // ---- the row tile's end.  1/l of every row through LDS; then the results, 64 rows x 1024 bytes, through the idle tile memory: 16-byte
        // piece i of row j at i ^ (j & 31), and out a row per store.  A piece's sums go out as they lie in registers.
        l_run = quarters_sum(l_run);
        float *const sums = reinterpret_cast<float *>(pool + MAX_AT), *const il = reinterpret_cast<float *>(pool + ALPHA_AT);
        __syncthreads();
        if (l < 16) sums[64 * kh + 16 * hq + l16] = l_run;
        __syncthreads();
        if (kh == 0 && l < 16) {
            const int r = 16 * hq + l16;
            const float sum = sums[r] + sums[64 + r];
            il[r] = sum == 0.f ? 0.f : 1.0f / sum;         // a row that sees no key is zeros
            if (!whole) {
                const f32x2 ml = {m_run, sum};
                *reinterpret_cast<f32x2 *>(p.part_ml + ((long long)piece * LA_ROWS + r) * 2) = ml;
            } else if (p.lse && row0 + r < rows) {
                p.lse[(long long)at.q0 * p.heads + row0 + r] = sum == 0.f ? -INFINITY : (m_run + __builtin_amdgcn_logf(sum)) * 0.693147180559945f;
            }
        }
        if (!whole) {
            float *const dst = p.part_o + (long long)piece * PIECE + ((w * 16) * 64 + l) * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    *reinterpret_cast<f32x4 *>(dst + (4 * i + q4) * 256) = f32x4{o[i][4 * q4], o[i][4 * q4 + 1], o[i][4 * q4 + 2], o[i][4 * q4 + 3]};
        } else {
            __syncthreads();
#pragma unroll
            for (int hb = 0; hb < 2; ++hb) {
                const float iv = il[32 * hb + col];
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        const f32x16 &a = o[2 * hb + d];
                        const u32x2 pk = {pack_bf16x2(a[4 * q4] * iv, a[4 * q4 + 1] * iv), pack_bf16x2(a[4 * q4 + 2] * iv, a[4 * q4 + 3] * iv)};
                        const int chunk = 32 * (w & 1) + 4 * (4 * d + q4) + (w >> 1);            // of the row, in channel order
                        *reinterpret_cast<u32x2 *>(pool + (32 * hb + col) * (DN * 2) + 16 * (chunk ^ col) + 8 * half) = pk;
                    }
            }
            __syncthreads();
            u32x4 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const u32x4 *>(pool + (8 * w + e) * (DN * 2) + 16 * (l ^ ((8 * w + e) & 31)));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = row0 + 8 * w + e;
                if (r < rows) {
                    const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                    *reinterpret_cast<u32x4_a2 *>(p.out + (long long)(at.q0 + tok) * p.o_t + (long long)head * p.o_h + 8 * l) = v[e];
                }
            }
        }
        __syncthreads();                                   // (the next row tile's queries go over these)
        u = want = to;
        first_segment = false;
        if (u >= u_end) break;
    }
    if (!p.by_tile && tid == 0 && !said) p.joins[4 * blockIdx.x + 1] = 0;
}

// The pieces of row tiles that workgroups share: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in the order of the keys.  A workgroup
// joins block i of wave w's channels (as the attention kernel's registers have them) of an entry's rows, four 16-byte values to a lane, its four
// waves a quarter of the pieces each.
__global__ __launch_bounds__(256) void latent_join_kernel(const LaParams p)
{
    __shared__ f32x4 sums[3][4][64];
    __shared__ float stats[3][2][32];
    const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = l >> 5, col = l & 31;
    const int32_t *const join = p.joins + 4 * (blockIdx.x >> 5);
    const int n = join[1];
    if (n <= 1) return;
    const int first = join[0], row0 = join[2], rows = join[3];
    const int w = (blockIdx.x & 31) >> 2, i = blockIdx.x & 3, hb = i >> 1, d = i & 1;
    // where the pieces are: that of the first workgroup is said; the others' ranges begin inside the row tile, so it is their first
    const int g = first >> 1;
    auto place = [&](const int k) { return (long long)(k == 0 ? first : 2 * (g + k)); };
    float top = LOW, total = 0.f;
    f32x4 acc[4];
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) acc[q4] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = wave; k < n; k += 4) {
        const f32x2 ml = *reinterpret_cast<const f32x2 *>(p.part_ml + (place(k) * LA_ROWS + 32 * hb + col) * 2);
        const float *src = p.part_o + place(k) * PIECE + ((w * 16 + 4 * i) * 64 + l) * 4;
        f32x4 x[4];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) x[q4] = *reinterpret_cast<const f32x4 *>(src + q4 * 256);
        const float m = fmaxf(top, ml[0]), a = __builtin_amdgcn_exp2f(top - m), b = __builtin_amdgcn_exp2f(ml[0] - m);
        top = m;
        total = total * a + ml[1] * b;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) acc[q4] = acc[q4] * a + x[q4] * b;
    }
    if (wave > 0) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) sums[wave - 1][q4][l] = acc[q4];
        if (half == 0) stats[wave - 1][0][col] = top, stats[wave - 1][1][col] = total;
    }
    __syncthreads();
    if (wave > 0) return;
    for (int k = 0; k < 3; ++k) {
        const float mk = stats[k][0][col], m = fmaxf(top, mk), a = __builtin_amdgcn_exp2f(top - m), b = __builtin_amdgcn_exp2f(mk - m);
        top = m;
        total = total * a + stats[k][1][col] * b;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) acc[q4] = acc[q4] * a + sums[k][q4][l] * b;
    }
    const int row = 32 * hb + col;
    if (row >= rows) return;
    const long long r = (long long)row0 + row;
    if (p.lse && w == 0 && d == 0 && half == 0) p.lse[r] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.693147180559945f;
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    const int tok = divide((int)r, p.of_heads), head = (int)r - tok * p.heads;
    uint16_t *dst = p.out + (long long)tok * p.o_t + (long long)head * p.o_h;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
        const int chunk = 32 * (w & 1) + 4 * (4 * d + q4) + (w >> 1);
        *reinterpret_cast<u32x2_a2 *>(dst + 8 * chunk + 4 * half) =
            u32x2{pack_bf16x2(acc[q4][0] * inv, acc[q4][1] * inv), pack_bf16x2(acc[q4][2] * inv, acc[q4][3] * inv)};
    }
}

}  // namespace

hipError_t latent_attention_launch(const LaParams &p, hipStream_t stream)
{
    if (p.bs % 4 == 0 && p.cache.rows % 4 == 0) hipLaunchKernelGGL((latent_attention_kernel<true>), dim3((unsigned)p.groups), dim3(THREADS), 0, stream, p);
    else hipLaunchKernelGGL((latent_attention_kernel<false>), dim3((unsigned)p.groups), dim3(THREADS), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(latent_join_kernel, dim3((unsigned)p.entries * 32), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pto
