// Launch parameters of the operators around a prompt: rotary positions, cache write and read, prompt attention
// (internal to the library).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pto {

// ---- rotary positions (rotary_kernels.hip)

constexpr int ROT_MAX_PAIRS = 128;

struct RotaryTablesParams {
    const void *positions;    // [T] int64 or int32
    const double *freq;       // [pairs] radians per position
    void *cos, *sin;          // [T, 2 * pairs], both halves alike
    long long T;
    int pairs, wide, dtype;   // wide: positions are int64
    float factor;
};
hipError_t rotary_tables_launch(const RotaryTablesParams &p, hipStream_t stream);

struct RotarySide {           // the queries or the keys: [T, heads, dim]
    const void *in;
    void *out;
    int heads, dim, offset;   // channels offset .. offset + 2 * pairs - 1 turn, the others are copied (in place: left alone)
    int copies;               // out is not in, and there are other channels
    long long in_t, in_h, out_t, out_h;   // strides in elements
    int parts;                // workgroups that share a token's heads (set by rotary_launch)
};
struct RotaryParams {
    RotarySide side[2];       // queries, keys (heads 0: none)
    const void *positions;
    const double *freq;
    long long T;
    int pairs, wide, dtype, layout;
    float factor;
    int cus;                              // compute units
    int tokens;                           // of a workgroup (set by rotary_launch)
};
hipError_t rotary_launch(const RotaryParams &p, hipStream_t stream);

// ---- the latent cache (latent_cache_kernels.hip)

struct CacheRows {            // the three parts of a cache row, each with its own base and row pitch in bytes
    uint8_t *nope, *rope, *scale;
    int nope_pitch, rope_pitch, scale_pitch;
    long long rows;
};
struct CacheWriteParams {
    const void *latent, *rope;            // [T, 512], [T, 64]
    long long latent_t, rope_t;           // strides in elements
    const long long *index;               // [T]
    CacheRows cache;
    uint16_t *values;                     // [T, 512] bf16 or null
    long long values_t;
    long long T;
    int dtype;
    int one_rounding;                     // 127 / max in one rounding
};
hipError_t cache_write_launch(const CacheWriteParams &p, hipStream_t stream);

struct CacheReadParams {
    CacheRows cache;
    const int32_t *bt;                    // [B, maxblk]
    const int32_t *cu;                    // [B + 1]
    const int32_t *first;                 // [B] or null
    uint16_t *latent, *rope;              // [rows, 512], [rows, 64] bf16
    long long latent_t, rope_t;           // strides in elements
    long long rows;                       // of the outputs
    int B, maxblk, bs;
};
hipError_t cache_read_launch(const CacheReadParams &p, hipStream_t stream);

// ---- prompt attention (prompt_attention.hip)

constexpr int PA_KEYS = 64;               // keys of a tile
constexpr int PA_WAVE_ROWS = 32;
constexpr int PA_MAX_SPLITS = 128;

struct PaParams {
    const uint16_t *q, *qr, *k, *kr, *v;
    uint16_t *out;
    float *lse;                           // [total_q, heads] or null
    float *part_o, *part_ml;              // [row][split][d], [row][split][2] of split rows
    const int32_t *cu_q, *cu_k;
    long long q_t, q_h, qr_t, qr_h, k_t, k_h, kr_t, kr_h, v_t, v_h, o_t, o_h;   // strides in elements
    long long total_q, total_k;
    int B, kv_heads, group, d, rope, fp16, causal;
    int window, sinks;                    // keys up to its own that a row sees, and first ones (window 0: all up to its own)
    int most_tiles;                       // most tiles of keys that a row tile of such a window sees
    int q_whole;                          // queries come in whole 16-byte pieces
    int splits, split_tiles;              // most splits of a row tile's keys; tiles from which a further split begins
    int waves;                            // of a workgroup, PA_WAVE_ROWS rows each: 8, or 4
    int grid;                             // workgroups, a multiple of eight
    int cus;                              // compute units
    float scale_log2;
};
hipError_t prompt_attention_launch(const PaParams &p, hipStream_t stream);

// pieces that a sequence's keys are divided into
__host__ __device__ inline int pa_splits_of(const int key_tiles, const int split_tiles, const int most)
{
    const int n = (key_tiles + split_tiles - 1) / split_tiles;
    return n < 1 ? 1 : (n > most ? most : n);
}

// tiles of a sequence's keys, as far as a row tile sees them
__host__ __device__ inline int pa_tiles_of(const int keys, const int most)
{
    const int n = (keys + PA_KEYS - 1) / PA_KEYS;
    return n < most ? n : most;
}

}  // namespace pto
