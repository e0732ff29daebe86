// What the two kernels of the attention over cached latents share: the line of work and its division, what a row tile sees, cache rows.
#pragma once
#include <type_traits>

#include "common.h"
#include "serving_ops.h"

namespace pto {
namespace {

constexpr int DN = 512, DR = 64;
constexpr int KT = LA_KEYS;
constexpr int PITCH = (DN + DR + 8) * 2;                  // bytes of a tile row: 512 latent and 64 rope channels as bf16, 16 spare
constexpr int TILE = KT * PITCH;
constexpr float TAU = 8.0f;                               // log2 units: the reference maximum moves only when exceeded by 2^8
constexpr float LOW = -1.7e38f;                           // reference maximum of a row that has seen no key yet

__device__ const u32x4 no_page[8 * (DN + 2 * DR + 16) / 16] = {};      // what eight keys without a page read, a whole row of the cache each

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
// int8 times the scale as bf16, each product rounded to fp32 and then to bf16: of a dword's lower and upper two
__device__ __forceinline__ uint32_t dequant_lower(const uint32_t r, const float sc)
{
    float f0, f1;
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f0) : "v"(r));
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f1) : "v"(r));
    return pack_bf16x2(f0 * sc, f1 * sc);
}
__device__ __forceinline__ uint32_t dequant_upper(const uint32_t r, const float sc)
{
    float f0, f1;
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f0) : "v"(r));
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f1) : "v"(r));
    return pack_bf16x2(f0 * sc, f1 * sc);
}
__device__ __forceinline__ u32x2 dequant_dword(const uint32_t r, const float sc) { return u32x2{dequant_lower(r, sc), dequant_upper(r, sc)}; }

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

// A sequence as the kernels take it: whatever the tables say, inside the tensors.
struct Sequence {
    int q0, n, keys;                                       // first token, tokens, keys
    int tiles, row_tiles;                                  // units of a row tile but LA_OPEN; row tiles
};
template <int ROWS>
__device__ __forceinline__ void count_tiles(const LaParams &p, Sequence &c)
{
    c.row_tiles = (c.n * p.heads + ROWS - 1) / ROWS;
    c.tiles = la_tiles_of(c.keys);
    c.tiles = c.tiles < p.most_tiles ? c.tiles : p.most_tiles;
}
template <int ROWS>
__device__ __forceinline__ Sequence sequence(const LaParams &p, const int b)
{
    Sequence c;
    const int total = (int)p.total_q;
    int lo = p.cu_q[b], hi = p.cu_q[b + 1], keys = p.lens[b];
    lo = lo < 0 ? 0 : (lo > total ? total : lo);
    hi = hi < lo ? lo : (hi > total ? total : hi);
    keys = keys < 0 ? 0 : (keys > p.most_keys ? p.most_keys : keys);
    c.q0 = lo, c.n = hi - lo, c.keys = keys;
    count_tiles<ROWS>(p, c);
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

// A boundary `x` units into a row tile of `len`, moved to its edge where a piece of one tile would be left (where three would be, neighbours that get them end
// last: single tokens of 32 sequences over 2052 keys 50.4 us, so 47.7).
constexpr int NEAR_BEGIN = LA_OPEN + 1, NEAR_END = 1;
__device__ __forceinline__ int moved(const int x, const int len) { return x <= NEAR_BEGIN ? 0 : (x >= len - NEAR_END ? len : x); }

// Units and row tiles of the sequences up to each: an entry to a thread, of as many sequences as that takes.  And what is kept here while a row
// tile's keys are gone through, since scalar registers are few: the line, this workgroup's part of it, the row tile in hand.
template <int THREADS>
struct LineTable {
    long long upto[THREADS], of_waves[THREADS / 64];
    long long tiles_of_waves[THREADS / 64], wide_of_waves[THREADS / 64];
    int tiles_upto[THREADS];
    int q0[THREADS], n[THREADS], keys[THREADS];            // of an entry's first sequence
    long long units, share, end, next;                     // end: of this workgroup's part; next: the unit behind the row tile's part in hand
    int groups, g, rest, said;
    Place place;                                           // the row tile in hand, or (fresh) the one that begins this workgroup's part
    int fresh, whole, piece;                               // whole: no other workgroup has a part of it; its piece's place
};

// The line of all units, and this workgroup's part of it.  CHOOSE: the call may be that of the other form, of LA_WIDE_ROWS.
template <int ROWS, int THREADS, bool CHOOSE>
struct Line {
    const LaParams &p;
    LineTable<THREADS> &t;

    __device__ __forceinline__ Line(const LaParams &params, LineTable<THREADS> &table) : p(params), t(table) {}

    static __device__ __forceinline__ int one(const int &x) { return __builtin_amdgcn_readfirstlane(x); }

    // Counts the sequences; false: this workgroup does not take part.
    __device__ __forceinline__ bool begin() const
    {
        const int tid = threadIdx.x, w = tid >> 6;
        long long mine = 0, tiles = 0, wide = 0;           // wide: tiles, if rows came by LA_WIDE_ROWS
        for (int j = 0; j < p.per_entry; ++j) {
            const int b = tid * p.per_entry + j;
            if (b < p.B) {
                const Sequence c = sequence<ROWS>(p, b);
                if (j == 0) t.q0[tid] = c.q0, t.n[tid] = c.n, t.keys[tid] = c.keys;
                mine += (long long)c.row_tiles * (c.tiles + LA_OPEN), tiles += c.row_tiles;
                if (CHOOSE) wide += (long long)((c.n * p.heads + LA_WIDE_ROWS - 1) / LA_WIDE_ROWS) * c.tiles;
            }
        }
        mine = wave_sums(mine);
        tiles = wave_sums(tiles);
        if (CHOOSE) wide = wave_sums(wide);
        if ((tid & 63) == 63) {
            t.of_waves[w] = mine, t.tiles_of_waves[w] = tiles;
            if (CHOOSE) t.wide_of_waves[w] = wide;
        }
        __syncthreads();
        for (int i = 0; i < w; ++i) mine += t.of_waves[i], tiles += t.tiles_of_waves[i];
        t.upto[tid] = mine;
        t.tiles_upto[tid] = tiles <= p.most_row_tiles ? (int)tiles : -1;
        __syncthreads();
        // (sequences that overlap, of beginnings that do not ascend, may be more than there are rows and joins for: then nothing is done)
        const int all_tiles = one(t.tiles_upto[THREADS - 1]);
        const long long units = all_tiles < 0 ? 0 : first_of(t.upto[THREADS - 1]);
        if (CHOOSE) {                                      // is the call the other form's?  (see latent_plan)
            const long long here = units - (long long)LA_OPEN * all_tiles;
            wide = 0;
            for (int i = 0; i < THREADS / 64; ++i) wide += first_of(t.wide_of_waves[i]);
            const bool leave = (here >= p.wide_tiles || all_tiles >= p.wide_row_tiles) && 16 * wide <= 9 * here;
            if (blockIdx.x == 0 && tid == 0) *p.form = leave;
            if (leave) return false;
        }
        // workgroups that take part, so that none gets less than LA_LEAST units
        const int pieces = units < (long long)p.groups * LA_LEAST ? (int)units / LA_LEAST : p.groups, groups = pieces > 0 ? pieces : 1;
        const int per_xcd = (groups + 7) / 8, slot = blockIdx.x >> 3, g = (int)(blockIdx.x & 7) * per_xcd + slot;
        const bool there = slot < per_xcd && g < groups && units > 0;
        if (tid == 0) {
            // Which row tiles are joined, and from how many pieces, is said by the workgroup that has the first of them; for every other entry that
            // there are none
            if (p.by_tile) {
                for (int i = (all_tiles < 0 ? 0 : all_tiles) + (int)blockIdx.x; i < p.entries; i += (int)gridDim.x) p.joins[4 * i + 1] = 0;
            } else if (!there) {
                p.joins[4 * blockIdx.x + 1] = 0;
            }
        }
        if (!there) return false;
        // the line's even divisions: units * i / groups
        long long share = (long long)((double)units / (double)groups);
        if (share * groups > units) --share;
        const int rest = (int)(units - share * groups);
        // (half of the waves look for this workgroup's end, the others for its beginning; each value is written by several threads alike)
        t.units = units, t.share = share, t.groups = groups, t.rest = rest, t.g = g;
        if (tid == 0) t.said = 0;
        const int upper = __builtin_amdgcn_readfirstlane(tid >= THREADS / 2);
        const long long u = division(share, rest, groups, g + upper < groups ? g + upper : g);
        const Place at = place_of(u);
        const int len = at.tiles + LA_OPEN, x = moved((int)(u - at.begin), len);
        if (upper) t.end = g + 1 < groups ? at.begin + x : units;
        else t.next = at.begin + x, t.place = at, t.fresh = x < len ? 1 : 0;
        __syncthreads();
        return true;
    }
    __device__ __forceinline__ static long long division(const long long share, const int rest, const int groups, const int i) { return share * i + (rest * i) / groups; }
    // the row tile that unit u of the line is in
    __device__ __forceinline__ Place place_of(const long long u) const
    {
        const int entries = p.seq_entries;
        int e = 0;                                         // entries that end in front of u
        for (int i = 0; i < entries; i += 64) e += __popcll(__ballot(t.upto[i + (threadIdx.x & 63)] <= u));
        long long first = e > 0 ? first_of(t.upto[e - 1]) : 0;
        int tiles_before = e > 0 ? one(t.tiles_upto[e - 1]) : 0;
        Place at;
        at.b = e * p.per_entry;
        Sequence c;
        c.q0 = one(t.q0[e]), c.n = one(t.n[e]), c.keys = one(t.keys[e]);
        count_tiles<ROWS>(p, c);
        for (int j = 1; j < p.per_entry; ++j) {            // (only of more sequences than threads)
            const long long next = first + (long long)c.row_tiles * (c.tiles + LA_OPEN);
            if (next > u || at.b + 1 >= p.B) break;
            first = next, tiles_before += c.row_tiles, ++at.b;
            c = sequence<ROWS>(p, at.b);
        }
        at.q0 = c.q0, at.n = c.n, at.keys = c.keys, at.tiles = c.tiles;
        at.row_tile = one(quotient(u - first, c.tiles + LA_OPEN));
        at.ordinal = tiles_before + at.row_tile;
        at.begin = first + (long long)at.row_tile * (c.tiles + LA_OPEN);
        return at;
    }

    // The next row tile of this workgroup's part, and the range of its tiles that are in it; false: there is none.  Between two calls there has
    // to be a barrier.
    __device__ __forceinline__ bool next(Place &at, int &i_begin, int &i_end) const
    {
        const long long u = first_of(t.next), u_end = first_of(t.end);
        if (u >= u_end) return false;
        const int fresh = one(t.fresh);                    // 1: the place is that of u, which nothing of was done; 0: that of something else; -1: of the row tile in front
        const bool first_part = fresh >= 0;
        at.b = one(t.place.b), at.q0 = one(t.place.q0), at.n = one(t.place.n), at.keys = one(t.place.keys), at.tiles = one(t.place.tiles);
        at.row_tile = one(t.place.row_tile), at.ordinal = one(t.place.ordinal), at.begin = first_of(t.place.begin);
        if (fresh < 0 && (at.row_tile + 1) * ROWS < at.n * p.heads) ++at.row_tile, ++at.ordinal, at.begin = u;
        else if (fresh <= 0) at = place_of(u);
        const int len = at.tiles + LA_OPEN;
        const long long end = at.begin + len, to = u_end < end ? u_end : end;
        const bool whole = u == at.begin && to == end;
        i_begin = (int)(u - at.begin) - LA_OPEN;
        i_begin = i_begin < 0 ? 0 : i_begin;
        i_end = (int)(to - at.begin) - LA_OPEN;
        const int groups = one(t.groups), g = one(t.g), piece = 2 * g + (first_part ? 0 : 1), rows = at.n * p.heads, row0 = at.row_tile * ROWS;
        if (threadIdx.x == 0 && u == at.begin && (p.by_tile || !whole)) {
            int n = 0;
            if (!whole) {                                  // pieces: one more than there are boundaries inside, those before unit `edge`
                const long long units = first_of(t.units), share = first_of(t.share), edge = end - NEAR_END;
                const int rest = one(t.rest);
                n = (int)((double)edge * (double)groups / (double)units) - g;
                n = n > 1 ? n - 1 : 1;
                while (g + n < groups && division(share, rest, groups, g + n) < edge) ++n;
            }
            int32_t *const join = p.joins + 4 * (p.by_tile ? at.ordinal : (int)blockIdx.x);
            join[0] = piece, join[1] = n, join[2] = at.q0 * p.heads + row0, join[3] = rows - row0 < ROWS ? rows - row0 : ROWS;
            t.said = 1;
        }
        __syncthreads();                                   // (everyone has read what is written now)
        t.next = to, t.whole = whole, t.piece = piece, t.place = at, t.fresh = -1;
        return true;
    }
    __device__ __forceinline__ void done() const
    {
        if (threadIdx.x == 0 && !p.by_tile && !t.said) p.joins[4 * blockIdx.x + 1] = 0;
    }
};

// What a row tile's tokens see, and which of its units are which tiles of keys: those of the first keys, then those that windows reach.
template <int ROWS>
struct Sight {
    const LaParams &p;
    int rows, row0, last, n, keys;                         // of the sequence; the row tile's first row, its last one's number in it
    int context;                                           // keys before the tree (below zero: as many of its first nodes have no key)
    int least, most, low_last;                             // keys that all, that some rows see (but for windows); where the last row's window begins
    int sink_tiles, skip, tiles;

    __device__ __forceinline__ Sight(const LaParams &params, const Place &at) : p(params)
    {
        rows = at.n * p.heads, row0 = at.row_tile * ROWS, n = at.n, keys = at.keys;
        last = rows - 1 - row0 < ROWS - 1 ? rows - 1 - row0 : ROWS - 1;
        const int tok0 = divide(row0, p.of_heads), tok1 = divide(row0 + last, p.of_heads);
        context = keys - n;
        least = !p.mask ? sees(tok0) : (context > 0 ? context : 0), most = sees(tok1);
        const int low = from(sees(tok0)) / KT;
        low_last = from(sees(tok1));
        sink_tiles = (p.sinks + KT - 1) / KT;
        sink_tiles = sink_tiles < low ? sink_tiles : low;
        skip = low - sink_tiles;
        tiles = la_tiles_of(most) - skip;
    }
    __device__ __forceinline__ int sees(const int tok) const
    {
        const int s = keys - n + tok + 1;
        return p.mask ? keys : (s < 0 ? 0 : s);
    }
    __device__ __forceinline__ int from(const int s) const { return p.window > 0 && s > p.window ? s - p.window : 0; }
    // (without a sign: a tile asked for ahead may lie behind the last key, and past 2^31)
    __device__ __forceinline__ uint32_t first_key(const int i) const { return (uint32_t)KT * (uint32_t)(i < sink_tiles ? i : i + skip); }
    // whether all rows see all 32 keys from this one on
    __device__ __forceinline__ bool whole(const uint32_t first) const
    {
        return first + KT <= (uint32_t)least && (first >= (uint32_t)low_last || first + KT <= (uint32_t)p.sinks);
    }
    // Bit i: whether a row that sees `s` keys (with this mask, if there is one) sees key first + i.
    __device__ __forceinline__ uint32_t seen(const uint32_t first_key, const int s, const unsigned long long *mask) const
    {
        const int first = (int)first_key;                  // (of a tile that has keys)
        auto below = [](int x) {
            x = x < 0 ? 0 : (x > 32 ? 32 : x);
            return (uint32_t)((1ull << x) - 1);
        };
        const int sinks = p.sinks < s ? p.sinks : s;
        uint32_t bits = (below(s - first) & ~below(from(s) - first)) | below(sinks - first);
        if (mask && (context < 0 || first_key + KT > (uint32_t)context)) {       // of the tile's keys, those in front of the tree and those of it that the mask names
            const int node = first - context, at_word = node >> 6, shift = node & 63;
            auto word = [&](const int i) { return i < 0 ? ~0ull : (i < p.words ? mask[i] : 0ull); };
            const unsigned long long lo = word(at_word), hi = word(at_word + 1);
            bits &= (uint32_t)((lo >> shift) | (shift ? hi << (64 - shift) : 0ull));
        }
        return bits;
    }
};

// A scale that is no number, or with which 127 steps are not finite, would be in the sums of rows that do not see the key (0 times it):
// such a group's values become zeros and the key's rope channels, which are in scores alone, no numbers.  A row that sees the
// key is then no number, others are not touched.  LANES neighbouring lanes hold a key.
// (Without a branch, around which registers would move.)
template <int LANES, typename Rope>
__device__ __forceinline__ void check_scale(float &scale, Rope &rope)
{
    const bool bad = !(fabsf(scale) < 2.6e36f);
    const uint64_t any = __ballot(bad);
    scale = bad ? 0.f : scale;
    const bool key_bad = ((uint32_t)(any >> ((threadIdx.x & 63) & ~(LANES - 1))) & ((1u << LANES) - 1)) != 0;
#pragma unroll
    for (unsigned i = 0; i < sizeof(Rope) / 4; ++i) rope[i] = key_bad ? 0x7fc07fc0u : rope[i];
}

// Where keys are in the cache.  NEAR: pages and the cache hold whole groups of NEAR rows, so one scalar look-up and one address serve NEAR
// neighbouring keys (from a multiple of NEAR on); those past the sequence's last one are what is left of the group in its page: their scores
// are hidden, and check_scale keeps what they hold out of the sums.  NEAR 1: each lane looks its own key up, and keys past the last stand
// in with it.
struct Page {
    int page, within;
};
struct RowAt {
    const uint8_t *nope, *scale, *rope;
};
template <int NEAR>
__device__ __forceinline__ Page page_of(const LaParams &p, const Place &at, const uint32_t asked)
{
    const uint32_t last = NEAR > 1 ? (at.keys - 1) & ~(NEAR - 1) : at.keys - 1;
    const int key = (int)(asked < last ? asked : last);
    const int block = divide(key, p.of_bs);                // (the block table has it: at.keys is no more than its pages hold)
    const int32_t *const entry = p.bt + (long long)at.b * p.maxblk + block;
    return Page{NEAR > 1 ? constant<int32_t>(entry) : *entry, key - block * p.bs};
}
__device__ __forceinline__ RowAt row_at(const LaParams &p, const Page k)
{
    const long long row = (long long)k.page * p.bs + k.within;
    const bool there = k.page >= 0 && row < p.cache.rows;
    // (without branches)
    const uint64_t yes = there ? ~0ull : 0ull, none = reinterpret_cast<uint64_t>(no_page) & ~yes;
    auto at = [&](const uint8_t *base, const int pitch) {
        return reinterpret_cast<const uint8_t *>(((reinterpret_cast<uint64_t>(base) + (uint64_t)row * (uint64_t)pitch) & yes) | none);
    };
    return {at(p.cache.nope, p.cache.nope_pitch), at(p.cache.scale, p.cache.scale_pitch), at(p.cache.rope, p.cache.rope_pitch)};
}

}  // namespace
}  // namespace pto
