// Launch parameters of a serving step's operators: pages and slots of the cache, attention over the cached latents
// (internal to the library).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "prompt_ops.h"

namespace pto {

// n / d for 0 <= n < 2^31 by a product: (high half of n * magic + n) >> shift, magic = floor(2^32 (2^shift - d) / d) + 1 for the
// smallest 2^shift >= d
struct Divisor {
    uint32_t magic;
    int shift;
};
inline Divisor divisor_of(const uint32_t d)
{
    int shift = 0;
    while ((1ull << shift) < d) ++shift;
    return {(uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1), shift};
}
__device__ __forceinline__ int divide(const int n, const Divisor d) { return (int)((__umulhi((uint32_t)n, d.magic) + (uint32_t)n) >> d.shift); }

// ---- pages and slots (paged_layout.hip)

struct CachePagesParams {
    const int32_t *before, *after;        // [B]
    int32_t *bt;                          // [B, maxblk]
    int32_t *stack;                       // [room]
    const int32_t *count;                 // [1]
    int32_t *left;                        // [1], may be count
    long long room;
    int B, maxblk, bs;
};
hipError_t cache_pages_launch(const CachePagesParams &p, hipStream_t stream);

constexpr int SLOTS_MAX_WORDS = 16;
struct CacheSlotsParams {
    const int32_t *new_lens, *all_lens;   // [B]
    const int32_t *bt;                    // [B, maxblk]
    int32_t *cu_q, *cu_k;                 // [B + 1], cu_k or null
    long long *positions, *slots;         // [T]
    const int32_t *parents;               // [T] or null
    unsigned long long *mask;             // [T, words] or null
    long long T;
    int B, maxblk, bs, words;
    int cus;
};
hipError_t cache_slots_launch(const CacheSlotsParams &p, hipStream_t stream);

// ---- attention over the cached latents (latent_attention.hip)

constexpr int LA_ROWS = 64;               // (token, head) rows of a workgroup
constexpr int LA_KEYS = 32;               // keys of a tile
constexpr int LA_MOST_KEYS = 0x7ffffff0;  // of a sequence; the first key of a tile, of those asked for ahead too, is then a 32-bit number without a sign,
constexpr int LA_AHEAD = 4;               // and no more than this many tiles are asked for ahead
__host__ __device__ constexpr int la_tiles_of(const int keys) { return (int)(((uint32_t)keys + LA_KEYS - 1) / LA_KEYS); }
static_assert((uint64_t)LA_KEYS * (uint64_t)(la_tiles_of(LA_MOST_KEYS) + LA_AHEAD) + LA_KEYS < (1ull << 32) && la_tiles_of(LA_MOST_KEYS) == (1 << 26) && la_tiles_of(0) == 0,
              "no key number wraps");
constexpr int LA_OPEN = 6;                // what a row tile's beginning and end cost, in tiles
constexpr int LA_THREADS = 512;          // of a workgroup
constexpr int LA_WIDE_ROWS = 128, LA_WIDE_THREADS = 256;    // the same of the form for many rows
// Units of the shortest piece that the line is divided into.  Of 2, 4 and 6, us: one token with 128 heads over 500 keys 17.1, 19.5 and 22.9, over 3000 24.3, 23.0 and 24.3; a tree of 8
// tokens, 16 heads, over 2900 keys 23.4, 22.7 and 23.7; single tokens of 8 sequences over 1000, 16 heads, 25.2, 23.4 and 24.3; longer calls the same.
constexpr int LA_LEAST = 4;

struct LaParams {
    const uint16_t *q, *qr;               // [total_q, heads, 512], [total_q, heads, 64] bf16
    long long q_t, q_h, qr_t, qr_h, o_t, o_h;   // strides in elements
    CacheRows cache;
    const int32_t *bt;                    // [B, maxblk]
    const int32_t *cu_q;                  // [B + 1]
    const int32_t *lens;                  // [B]
    const unsigned long long *mask;       // [total_q, words] or null
    uint16_t *out;
    float *lse;                           // [total_q, heads] or null
    float *part_o, *part_ml;              // [2 * groups] pieces of a row tile: 512 sums a row, (maximum, sum) a row
    int32_t *joins;                       // [entries][4]: first piece, pieces, first row, rows
    long long total_q;
    int B, maxblk, bs, heads, words;
    int window, sinks;                    // window 0: all keys
    int most_keys, most_tiles;            // of a sequence, as the block table and the window have it
    int per_entry, seq_entries;           // sequences that a workgroup's thread counts; threads that count any
    int32_t *form;                        // [1]: whether the form of LA_WIDE_ROWS takes the call, which that of LA_ROWS says; null: the host did
    long long wide_tiles, wide_row_tiles; // ... from this many tiles or row tiles of LA_ROWS on
    int groups;                           // workgroups, a multiple of eight
    int most_row_tiles;                   // of sequences that do not overlap
    int by_tile, entries;                 // joins by row tile (of all sequences), else by workgroup; how many there are
    Divisor of_heads, of_bs;
    float scale_log2;
};
// by rows of LA_ROWS, of LA_WIDE_ROWS, or, both given, as the first finds right
hipError_t latent_attention_launch(const LaParams *narrow, const LaParams *wide, hipStream_t stream);
hipError_t latent_attention_wide_launch(const LaParams &p, hipStream_t stream);      // without the joining launch

}  // namespace pto
