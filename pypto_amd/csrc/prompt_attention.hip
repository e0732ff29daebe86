// Attention over whole prompts, gfx950: causal or not, grouped heads, packed sequences, keys that began before the queries.
//
// Row r of a key head's queries is (token r / G, head r % G of the group of G): a workgroup of W waves takes 32 * W consecutive rows of
// a sequence, so that all heads of a group share the keys that are read.  Per wave (32 rows) and tile of 64 keys:
//   S^T[key][row]  = K[key][:] . Q^T         v_mfma_f32_32x32x16, A = key rows from LDS, B = Q^T resident in registers
//   p = exp2(scale * s - m)                  one pass: running maximum and sum, fp32, a lane's keys of its own row
//   O^T[ch][row]  += V^T[ch][key] . P^T      A = V^T by the transposing LDS read, B = P^T straight from the accumulators:
// the accumulator of a 32x32 product gives lane (row, half) the keys 8 * (i / 4) + 4 * half + i % 4, and the transposing reads of
// V take keys in that order, so probabilities never leave their lane.  P is rounded to 16 bits un-normalised (what the matrix
// cores take); sums, maxima and outputs are fp32 until the last rounding.
//
// The rope part of queries and keys is a separate product over 64 more channels, whose keys all heads may share: nothing is
// concatenated in memory.
//
// Bound by the longer of a tile's two phases, which is the softmax and the requests.  32 rows and 64 keys of 128 + 64 channels are 1280 clocks of
// products to a wave, 2560 on a SIMD, whose two waves take turns; a tile takes 3250, two phases of 1625: 1080 clocks of softmax and 530 of
// requests of one half of the waves beside 1490 (the products and their operands' way) of the other.  Without rope parts 2900 for 2048 of
// products, phases of the same softmax and requests beside 1170.  4096 causal tokens of 128 heads, bf16: 637 to 690 us, 1080 to 1000 TFLOP/s of the
// products that the mask asks for; a product of 8192^3 reaches 1330.  Where its time goes (clocks read by two waves of each workgroup): 15 %
// of the compute units' time is without a workgroup, between two and at the launch's end, 11 % are workgroups' beginnings (11900 clocks) and ends (4250 of 127000),
// and of the 74 % in the loop products are 0.79: 0.58 in all, where the counters say 0.54, since of a sequence's last tiles some waves multiply
// nothing.  The shader clock is at 1.8 of 2.4 GHz meanwhile.  On the way: one phase, every wave products and softmax in turn 732 us; two
// phases, two stages of tiles, requests among the products 675; three stages, requests before the softmax 670 at fewer clocks; queries and
// results by whole cache lines 637.  Not kept: workgroups that stay and draw their work from counters (1 % slower here, 3 % faster for nine
// ragged sequences, 7 % slower where keys are divided).
#include <cmath>
#include <type_traits>

#include "common.h"
#include "prompt_device.h"
#include "prompt_ops.h"

namespace pto {
namespace {

constexpr float PA_TAU = 8.0f;            // log2 units: the reference maximum moves only when exceeded by 2^8
constexpr float PA_LOW = -1.7e38f;        // reference maximum of a row that has seen no key yet
constexpr int PA_ROPE = 64;

__device__ __forceinline__ void pa_barrier()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ float pa_other_max(const float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pa_other_sum(const float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

struct F16 {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x16 mfma(const frag a, const frag b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pack(const float lo, const float hi) { return pack_f16x2(lo, hi); }
};
struct BF16 {
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x16 mfma(const frag a, const frag b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint32_t pack(const float lo, const float hi) { return pack_bf16x2(lo, hi); }
};

__device__ __forceinline__ uint32_t opaque(uint32_t x)
{
    asm("" : "+v"(x));
    return x;
}
template <typename T>
__device__ __forceinline__ T lds_frag(const uint32_t at)
{
    return *(const __attribute__((address_space(3))) T *)(at);
}
__device__ __forceinline__ s16x4 lds_tr16(const uint32_t at) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(at)); }

// A sequence as the kernels take it: whatever the tables of beginnings say, inside the tensors.
struct Span {
    int begin, len;
};
__device__ __forceinline__ Span span_of(const int32_t *cu, const int b, const int total)
{
    int lo = cu[b], hi = cu[b + 1];
    lo = lo < 0 ? 0 : (lo > total ? total : lo);
    hi = hi < lo ? lo : (hi > total ? total : hi);
    return {lo, hi - lo};
}

// sums of x over this lane and all lanes before it
__device__ __forceinline__ int wave_sums(int x)
{
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);     // row_shr:1, 2, 4, 8: within rows of sixteen lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // row_bcast:15: rows 0 and 2 into 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // row_bcast:31: the lower half into the upper
    return x;
}

// Keys that local token t of a sequence sees.
__device__ __forceinline__ int pa_visible(const int t, const int lq, const int lk, const int causal)
{
    if (!causal) return lk;
    const int n = t + 1 + lk - lq;
    return n < 0 ? 0 : (n > lk ? lk : n);
}

// A tile in LDS.  Rows of 64 channels (eight 16-byte pieces) lie one behind the other, piece c of row r at c ^ (r / 2) % 8 (keys) or
// c ^ 4 * ((r / 2) % 2) (values).  Rows of 128 channels lie in blocks of four, 1040 bytes apart: [piece / 8][row][piece % 8], the last index ^ 4 in
// the lower two rows.  Then neither 16 lanes that read one piece of 16 key rows nor 16 lanes that read 32 value channels of four
// rows meet in a bank, and (128 channels) the pieces that a lane reads one after the other are constants away from one of two addresses.  A
// DMA request writes 1024 bytes in the order of its lanes, so the order of the pieces is in what each lane asks for; eight lanes ask for a
// whole cache line.  Where two workgroups with rope parts share a compute unit's 160 KiB there is no room between blocks: rows of 256 bytes, piece
// c of row r at c ^ r % 16 (keys) or c ^ 4 * (r % 4) (values), and an exclusive or to each read.
constexpr int PA_BLOCK = 1040;

// WINDOW: a row sees the last p.window of the keys up to its own, and the first p.sinks.  Tiles that no row of the workgroup sees, between
// the first keys and the windows, are stepped over: t counts the tiles that are left.  8192 tokens of 128 heads of 128 + 64 channels with a window of 1024: 812 to 820 us without first
// keys, 870 on the same machine with four (829 on another), as waves step over the tiles in front of their own windows only where no first keys stay visible.  Of a
// workgroup's 21 tiles its rows see 16 on average; per tile it takes what it does without windows.  Four waves, whose 128 rows need 19, took 841 for 829.
template <typename E, int D, int R, int W, bool WINDOW>
__global__ __launch_bounds__(64 * W, 2) void prompt_attention_kernel(const PaParams p)
{
    constexpr int ROWS = 32 * W;
    constexpr bool PHASED = W == 8;                        // two waves of a SIMD in this workgroup; otherwise of two workgroups
    constexpr int KP = D * 2;                              // bytes of a key row, and of a value row
    constexpr bool BLOCKS = D == 128 && !(R > 0 && W == 4), ROW_256 = D == 128 && !BLOCKS;    // how a tile lies in LDS
    constexpr int REQ = BLOCKS ? PA_BLOCK : 1024;          // bytes from one request's rows to the next one's
    constexpr int K_REQS = PA_KEYS * KP / 1024, R_REQS = PA_KEYS * R * 2 / 1024;
    constexpr int K_BYTES = K_REQS * REQ, R_BYTES = R_REQS * 1024;
    constexpr int K_STAGE = K_BYTES + R_BYTES;             // [keys | rope keys] of a tile
    constexpr int STAGES = PHASED ? 3 : 2, AHEAD = 5;
    constexpr int POOL = STAGES * (K_STAGE + K_BYTES) > W * 32 * 256 ? STAGES * (K_STAGE + K_BYTES) : W * 32 * 256;   // (results: 256 bytes to a row)
    constexpr int KS = D / 16, RS = R / 16, CT = D / 32;
    constexpr int NK = K_REQS / W, NR = R_REQS / W;   // requests of a wave per tile: keys (as many values), rope keys
    static_assert(K_REQS % W == 0 && R_REQS % W == 0, "whole requests for every wave");
    typedef typename E::frag frag;

    __shared__ __attribute__((aligned(1024))) uint8_t pool[POOL];   // keys of the stages' tiles, then their values

    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    // Items of work: (key head, sequence, row tile, piece of its keys), counted from the lengths.  An XCD takes consecutive ones, so that
    // workgroups which read the same head's keys share an L2; a sequence's last rows, which see the most keys, come first.
    struct Scan {                                          // of 64 sequences, one to a lane
        Span sq, sk;
        int tiles, splits, upto;                           // upto: items of a key head in this and all sequences before it (of these 64)
    };
    auto scan = [&](const int base) __attribute__((always_inline)) {
        Scan c;
        const int l = tid & 63, mine = base + l < p.B ? base + l : p.B - 1;
        c.sq = span_of(p.cu_q, mine, (int)p.total_q), c.sk = span_of(p.cu_k, mine, (int)p.total_k);
        c.tiles = base + l < p.B ? (c.sq.len * p.group + ROWS - 1) / ROWS : 0;
        c.splits = pa_splits_of(WINDOW ? pa_tiles_of(c.sk.len, p.most_tiles) : (c.sk.len + PA_KEYS - 1) / PA_KEYS, p.split_tiles, p.splits);
        c.upto = wave_sums(c.tiles * c.splits);
        return c;
    };
    Scan c = scan(0);
    int per_head = __builtin_amdgcn_readlane(c.upto, 63);
    for (int base = 64; base < p.B; base += 64) per_head += __builtin_amdgcn_readlane(scan(base).upto, 63);
    const int items = per_head * p.kv_heads, per_xcd = (items + 7) / 8, first = (blockIdx.x & 7) * per_xcd;
    const int here = items - first < per_xcd ? items - first : per_xcd;                     // items of this XCD
    for (int slot = blockIdx.x >> 3; slot < here; slot += gridDim.x >> 3) {
        // An XCD deals its workgroups to four groups of compute units in turn, whichever is free: every second four go backwards, so that
        // where a head has 4 n row tiles the same group does not get the longest of all of them (128 heads of 16 tiles 676 us, now 651).
        const int item = first + ((slot & 4) != 0 && (slot | 3) < here ? slot ^ 3 : slot);
        const int kvh = item / per_head;
        // (nothing that hangs on the lane alone is kept from one item to the next: it would take the registers of the products' operands)
        const int l = (int)opaque(tid & 63), n = l & 31, half = l >> 5;
        int rest = item - kvh * per_head, base = 0;
        while (rest >= __builtin_amdgcn_readlane(c.upto, 63)) {
            rest -= __builtin_amdgcn_readlane(c.upto, 63);
            base += 64;
            c = scan(base);
        }
        const int who = __builtin_ctzll(__ballot(c.upto > rest));
        rest -= who > 0 ? __builtin_amdgcn_readlane(c.upto, who - 1) : 0;
        const int lq = __builtin_amdgcn_readlane(c.sq.len, who), lk = __builtin_amdgcn_readlane(c.sk.len, who);
        const int q0 = __builtin_amdgcn_readlane(c.sq.begin, who), k0 = __builtin_amdgcn_readlane(c.sk.begin, who);
        const int splits = __builtin_amdgcn_readlane(c.splits, who);
        const int which = splits > 1 ? rest / splits : rest;
        const int split = rest - which * splits;
        const int tile = p.causal ? __builtin_amdgcn_readlane(c.tiles, who) - 1 - which : which;

        // This lane's row, and how many keys it sees.  Rows past the last one stand in with it and are never stored.
        const int rows = lq * p.group;
        const int row = tile * ROWS + 32 * w + n;
        const int row_in = row < rows ? row : rows - 1;
        const int tok = p.group > 1 ? row_in / p.group : row_in, head = kvh * p.group + row_in - tok * p.group;
        const int sees = pa_visible(tok, lq, lk, p.causal);
        const int last_row = tile * ROWS + ROWS - 1 < rows ? tile * ROWS + ROWS - 1 : rows - 1;
        const int wg_sees = pa_visible(last_row / p.group, lq, lk, p.causal);
        const int wave_most = tile * ROWS + 32 * w < rows ? pa_visible(__builtin_amdgcn_readlane(tok, 31), lq, lk, p.causal) : 0;
        const int wave_least = pa_visible(__builtin_amdgcn_readlane(tok, 0), lq, lk, p.causal);

        // where windows begin: of this lane's row, of the workgroup's first and the wave's last; tiles of the first keys in front of them, tiles
        // stepped over
        auto from_of = [&](const int n) { return WINDOW && n > p.window ? n - p.window : 0; };
        const int from = from_of(sees), wave_from = WINDOW ? from_of(wave_most) : 0;
        const int low = WINDOW ? from_of(pa_visible(tile * ROWS / p.group, lq, lk, 1)) / PA_KEYS : 0;
        const int sink_tiles = WINDOW ? ((p.sinks + PA_KEYS - 1) / PA_KEYS < low ? (p.sinks + PA_KEYS - 1) / PA_KEYS : low) : 0;
        const int skip = low - sink_tiles;
        auto tile_at = [&](const int t) { return WINDOW && t >= sink_tiles ? t + skip : t; };

        const int key_tiles = (wg_sees + PA_KEYS - 1) / PA_KEYS - skip;
        const int split_len = (key_tiles + splits - 1) / splits;
        const int t_begin = split * split_len;
        const int t_end = t_begin + split_len < key_tiles ? t_begin + split_len : key_tiles;

        // Requests of a tile: a wave's request brings 1024 bytes of whole rows.  Keys past the sequence's last one stand in with it (their
        // probabilities are zero, and what lies behind the sequence is never touched).
        const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte_t *)pool;
        const uint8_t *const k_base = reinterpret_cast<const uint8_t *>(p.k + k0 * p.k_t + kvh * p.k_h);
        const uint8_t *const v_base = reinterpret_cast<const uint8_t *>(p.v + k0 * p.v_t + kvh * p.v_h);
        const uint8_t *const r_base = R > 0 ? reinterpret_cast<const uint8_t *>(p.kr + k0 * p.kr_t + kvh * p.kr_h) : nullptr;
        constexpr int PER = 1024 / KP;                         // rows of a request
        const int row_of = BLOCKS ? (l >> 3) & 3 : l / (KP / 16);   // this lane's row of a request, and its pieces: of keys, values, rope keys
        const int k_piece = BLOCKS ? 8 * (l >> 5) + ((l & 7) ^ (4 * (row_of >> 1))) : ROW_256 ? (l & 15) ^ ((PER * w + row_of) & 15) : (l & 7) ^ (((PER * w + row_of) >> 1) & 7);
        const int v_piece = BLOCKS ? k_piece : ROW_256 ? (l & 15) ^ (4 * (row_of & 3)) : (l & 7) ^ (4 * ((row_of >> 1) & 1));
        const int r_piece = (l & 7) ^ (((8 * w + (l >> 3)) >> 1) & 7);
        static_assert(W % 2 == 0, "a wave's requests, W * 8 rows apart, have their pieces in the same places");
        const uint32_t k_off = (uint32_t)row_of * (uint32_t)(p.k_t * 2) + 16 * k_piece, v_off = (uint32_t)row_of * (uint32_t)(p.v_t * 2) + 16 * v_piece;
        const uint32_t r_off = (uint32_t)(l >> 3) * (uint32_t)(p.kr_t * 2) + 16 * r_piece;
        // the next tile's first row of this wave, of keys, rope keys and values, and which tiles these are
        const uint8_t *k_next = k_base + ((long long)tile_at(t_begin) * PA_KEYS + PER * w) * p.k_t * 2, *v_next = v_base + ((long long)tile_at(t_begin) * PA_KEYS + PER * w) * p.v_t * 2;
        const uint8_t *r_next = R > 0 ? r_base + ((long long)tile_at(t_begin) * PA_KEYS + 8 * w) * p.kr_t * 2 : nullptr;
        int k_tile = t_begin, v_tile = t_begin;
        // one request of a tile all of whose keys there are: NK of its keys, NR of its rope keys, NK of its values
        auto request_whole = [&](const int i, const int k_stage, const int v_stage) __attribute__((always_inline)) {
            if (i < NK) dma16_base(k_next + (long long)i * W * PER * p.k_t * 2, k_off, lds0 + k_stage * K_STAGE + (i * W + w) * REQ);
            else if (i < NK + NR) dma16_base(r_next + (long long)(i - NK) * W * 8 * p.kr_t * 2, r_off, lds0 + k_stage * K_STAGE + K_BYTES + ((i - NK) * W + w) * 1024);
            else dma16_base(v_next + (long long)(i - NK - NR) * W * PER * p.v_t * 2, v_off, lds0 + STAGES * K_STAGE + v_stage * K_BYTES + ((i - NK - NR) * W + w) * REQ);
        };
        // the requests of a sequence's last tile, from its last key on the same row again
        auto request_last = [&](const uint8_t *at, const long long pitch, const int piece, const int row_in, const uint32_t dst, const int left, const int i, const int each, const int bytes)
                                __attribute__((always_inline)) {
            const int r = (i * W + w) * each + row_in, from = r < left ? r : left - 1;
            dma16_base(at - (long long)each * w * pitch * 2, (uint32_t)from * (uint32_t)(pitch * 2) + 16 * piece, dst + (i * W + w) * bytes);
        };
        auto whole = [&](const int t) { return lk - tile_at(t) * PA_KEYS >= PA_KEYS; };
        auto next_keys = [&]() __attribute__((always_inline)) {
            k_next += PA_KEYS * 2 * p.k_t;
            if (R > 0) r_next += PA_KEYS * 2 * p.kr_t;
            ++k_tile;
            if (WINDOW && k_tile == sink_tiles) {
                k_next += (long long)skip * (PA_KEYS * 2) * p.k_t;
                if (R > 0) r_next += (long long)skip * (PA_KEYS * 2) * p.kr_t;
            }
        };
        auto next_values = [&]() __attribute__((always_inline)) {
            v_next += PA_KEYS * 2 * p.v_t;
            ++v_tile;
            if (WINDOW && v_tile == sink_tiles) v_next += (long long)skip * (PA_KEYS * 2) * p.v_t;
        };
        auto request_keys = [&](const int stage) __attribute__((always_inline)) {
            const int left = lk - tile_at(k_tile) * PA_KEYS;
            if (whole(k_tile)) {
#pragma unroll
                for (int i = 0; i < NK + NR; ++i) request_whole(i, stage, 0);
            } else {
#pragma unroll
                for (int i = 0; i < NK; ++i) request_last(k_next, p.k_t, k_piece, row_of, lds0 + stage * K_STAGE, left, i, PER, REQ);
#pragma unroll
                for (int i = 0; i < NR; ++i) request_last(r_next, p.kr_t, r_piece, l >> 3, lds0 + stage * K_STAGE + K_BYTES, left, i, 8, 1024);
            }
            next_keys();
        };
        auto request_values = [&](const int stage) __attribute__((always_inline)) {
            if (whole(v_tile)) {
#pragma unroll
                for (int i = 0; i < NK; ++i) request_whole(NK + NR + i, 0, stage);
            } else {
#pragma unroll
                for (int i = 0; i < NK; ++i) request_last(v_next, p.v_t, v_piece, row_of, lds0 + STAGES * K_STAGE + stage * K_BYTES, lk - tile_at(v_tile) * PA_KEYS, i, PER, REQ);
            }
            next_values();
        };

        // Queries into registers.  As the products want them a wave would ask for 32 bytes of each of its rows at a time; so they come through
        // LDS, whole cache lines to a request, into memory that later tiles use.  Queries that promise less than 16 bytes' alignment come
        // straight.
        frag qf[KS + RS];
        const long long q_at = (long long)(q0 + tok) * p.q_t + (long long)head * p.q_h, qr_at = R > 0 ? (long long)(q0 + tok) * p.qr_t + (long long)head * p.qr_h : 0;
        constexpr int Q_WAVE = 32 * (KP + 2 * R);
        static_assert(K_STAGE + W * Q_WAVE <= POOL, "the queries fit beside the first tile's keys");
        const uint32_t q_lds = lds0 + K_STAGE + w * Q_WAVE;
        auto of_row = [](const long long at, const int r) { return (long long)((uint64_t)(uint32_t)__shfl((int)at, r) | ((uint64_t)(uint32_t)__shfl((int)(at >> 32), r) << 32)); };
        auto request_queries = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 32 * KP / 1024; ++i) {
                const int r = i * PER + l / (KP / 16), piece = (l % (KP / 16)) ^ (D == 128 ? r & 15 : (r >> 1) & 7);
                dma16(p.q + of_row(q_at, r) + 8 * piece, q_lds + i * 1024);
            }
#pragma unroll
            for (int i = 0; i < 32 * 2 * R / 1024; ++i) {
                const int r = i * 8 + l / 8, piece = (l % 8) ^ ((r >> 1) & 7);
                dma16(p.qr + of_row(qr_at, r) + 8 * piece, q_lds + 32 * KP + i * 1024);
            }
        };
        auto read_queries = [&]() __attribute__((always_inline)) {
            if (p.q_whole) {
#pragma unroll
                for (int i = 0; i < KS; ++i) qf[i] = lds_frag<frag>(q_lds + n * KP + 16 * ((2 * i + half) ^ (D == 128 ? n & 15 : (n >> 1) & 7)));
#pragma unroll
                for (int i = 0; i < RS; ++i) qf[KS + i] = lds_frag<frag>(q_lds + 32 * KP + n * (2 * R) + 16 * ((2 * i + half) ^ ((n >> 1) & 7)));
            } else {
#pragma unroll
                for (int i = 0; i < KS; ++i) qf[i] = __builtin_bit_cast(frag, (u32x4) * reinterpret_cast<const u32x4_a2 *>(p.q + q_at + 8 * half + 16 * i));
#pragma unroll
                for (int i = 0; i < RS; ++i) qf[KS + i] = __builtin_bit_cast(frag, (u32x4) * reinterpret_cast<const u32x4_a2 *>(p.qr + qr_at + 8 * half + 16 * i));
            }
        };

        float scale = p.scale_log2;
        f32x16 o[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
        float m_run = PA_LOW, l_run = 0.f;                     // the row's reference maximum (log2), this lane's share of its sum

        // LDS addresses of the operand reads in stage 0: key row n, pieces 2 * ks + half; values: keys 4 * half + (l % 16) / 4 (+ 8), channels
        // 16 * ((l / 16) & 1) + 4 * (l % 4)
        constexpr int KA = BLOCKS ? 2 : ROW_256 ? 1 : KS, VA = ROW_256 ? 1 : 2;
        uint32_t k_lane[KA], r_lane[R > 0 ? RS : 1], v_lane[VA];
#pragma unroll
        for (int i = 0; i < KA; ++i)
            k_lane[i] = lds0 + (BLOCKS    ? (n >> 2) * REQ + (n & 3) * 128 + 16 * half + 64 * (i ^ ((n >> 1) & 1))
                                : ROW_256 ? n * KP + 16 * (half ^ (n & 15))
                                          : n * KP + 16 * ((2 * i + half) ^ ((n >> 1) & 7)));
#pragma unroll
        for (int i = 0; i < RS; ++i) r_lane[i] = lds0 + K_BYTES + n * (R * 2) + 16 * ((2 * i + half) ^ ((n >> 1) & 7));
        {
            const int row = (l & 15) >> 2, low = 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
#pragma unroll
            for (int i = 0; i < VA; ++i)
                v_lane[i] = lds0 + STAGES * K_STAGE + 8 * (l & 1) +
                            (BLOCKS    ? half * REQ + row * 128 + 64 * (i ^ (row >> 1)) + 16 * low
                             : ROW_256 ? (4 * half + row) * KP + 64 * row + 16 * low
                                       : (4 * half + row) * KP + 16 * ((4 * i + low) ^ (4 * (row >> 1))));
        }
        constexpr int V_EIGHT = BLOCKS ? 2 * REQ : 8 * KP;   // to the value row eight keys on

        f32x16 s[2];                                           // scores of the tile in hand
        frag pf[4];                                            // probabilities of the tile before it
        // The products of a tile: scores of the tile in one stage and, spread between them, the probabilities of the tile before it times its
        // values, in another; operands are read AHEAD products before their use.
        auto products = [&](auto with_scores, auto with_values, const int k_stage, const int v_stage) __attribute__((always_inline)) {
            constexpr int NQ = decltype(with_scores)::value ? 2 * (KS + RS) : 0, NP = decltype(with_values)::value ? 4 * CT : 0, N = NQ + NP;
            uint32_t kb[KA], rb[R > 0 ? RS : 1], vb[VA];        // (what the compiler cannot take apart: the rest of an address is an instruction's constant)
            if (NQ > 0) {
#pragma unroll
                for (int i = 0; i < KA; ++i) kb[i] = opaque(k_lane[i] + k_stage * K_STAGE);
#pragma unroll
                for (int i = 0; i < RS; ++i) rb[i] = opaque(r_lane[i] + k_stage * K_STAGE);
            }
            if (NP > 0) {
#pragma unroll
                for (int i = 0; i < VA; ++i) vb[i] = opaque(v_lane[i] + v_stage * K_BYTES);
            }
            frag a[N];
            auto is_value = [](const int j) { return (j + 1) * NP / N > j * NP / N; };
            auto read = [&](const int j) __attribute__((always_inline)) {
                const int pv = j * NP / N, qk = j - pv;        // products of either kind before this one
                if (is_value(j)) {
                    const int ks = pv / CT, c = pv % CT;
                    const uint32_t at = ROW_256 ? (vb[0] ^ (64 * c)) + 16 * ks * KP : vb[c & (VA - 1)] + (BLOCKS ? ks * 4 * REQ + (c >> 1) * 512 : 16 * ks * KP);
                    const s16x4 lo = lds_tr16(at), hi = lds_tr16(at + V_EIGHT);
                    a[j] = __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                } else {
                    const int h = qk & 1, i = qk >> 1;
                    a[j] = lds_frag<frag>(i >= KS   ? rb[(i - KS) % (R > 0 ? RS : 1)] + h * 32 * (R * 2)
                                          : BLOCKS  ? kb[(i >> 1) & (KA - 1)] + h * 8 * REQ + (i >> 2) * 512 + (i & 1) * 32
                                          : ROW_256 ? (kb[0] ^ (32 * i)) + h * 32 * KP
                                                    : kb[i % KA] + h * 32 * KP);
                }
            };
            const f32x16 zero = {};
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) read(j);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int pv = j * NP / N, qk = j - pv;
                if (is_value(j)) o[pv % CT] = E::mfma(a[j], pf[pv / CT], o[pv % CT]);
                else s[qk & 1] = E::mfma(a[j], qf[qk >> 1], qk < 2 ? zero : s[qk & 1]);
                __builtin_amdgcn_sched_barrier(0);
                if (j + AHEAD < N) read(j + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // The softmax of tile t: scores to probabilities.
        auto softmax = [&](const int count) __attribute__((always_inline)) {
            const int t = tile_at(count);
            if (WINDOW && ((t + 1) * PA_KEYS > wave_least || (t * PA_KEYS < wave_from && (t + 1) * PA_KEYS > p.sinks))) {
                // (without a branch for each score)
                const int first = t * PA_KEYS + 4 * half;
                if (t * PA_KEYS >= p.sinks) {
                    const uint32_t span = (uint32_t)(sees - from);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[h][i] = (uint32_t)(first - from + 32 * h + 8 * (i >> 2) + (i & 3)) < span ? s[h][i] : -INFINITY;
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int key = first + 32 * h + 8 * (i >> 2) + (i & 3);
                            const bool hidden = (key >= sees) | ((key < from) & (key >= p.sinks));
                            s[h][i] = hidden ? -INFINITY : s[h][i];
                        }
                }
            } else if (!WINDOW && (t + 1) * PA_KEYS > wave_least) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (t * PA_KEYS + 32 * h + 8 * (i >> 2) + 4 * half + (i & 3) >= sees) s[h][i] = -INFINITY;
            }
            float mx = s[0][0];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[h][i]);
            mx = pa_other_max(mx) * scale;
            if (__any(mx > m_run + PA_TAU)) {                  // rare: the reference follows the true maximum lazily
                const float m_new = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[c][i] *= alpha;
            }
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][8 * g + i], scale, -m_run));
                        sum[i & 1] += e[i];
                    }
                    const u32x4 pk = {E::pack(e[0], e[1]), E::pack(e[2], e[3]), E::pack(e[4], e[5]), E::pack(e[6], e[7])};
                    pf[2 * h + g] = __builtin_bit_cast(frag, pk);
                }
            l_run += sum[0] + sum[1];
        };

        // Two waves share a SIMD, and while one multiplies the other does the softmax of its tile.  Four waves to a workgroup: the other is of
        // another workgroup, and they find their turns themselves; a barrier ends a tile's products, behind it nobody reads the keys of tile t or
        // the values of tile t - 1, and those of tiles t + 2 and t + 1 are asked for.  Eight waves: the second half is one phase
        // behind, and a barrier ends every phase.  First half: phase 2t products of tile t (and t - 1), phase 2t + 1 its softmax.  A wave asks
        // for its part of the keys of tile t + 2 and the values of tile t + 1 where it has time, at the beginning of its softmax of tile t (in
        // phase 2t + 1 or 2t + 2: the last readers of those buffers, of the keys of tile t - 1 and the values of tile t - 2, were done with
        // phase 2t - 1), and waits for them at the end of its products of tile t + 1 (phase 2t + 2 or 2t + 3; the first reader's phase is
        // 2t + 4).  Asked for among the products they held up the first half's by 550 of 2050 clocks.
        const bool late = PHASED && w >= W / 2;
        const std::integral_constant<bool, true> yes;
        const std::integral_constant<bool, false> no;
        if (t_begin < t_end) {
            int s0 = 0, s1 = 1, s2 = PHASED ? 2 : 1;           // stages of tiles t, t + 1 and t - 1
            auto end_products = [&]() __attribute__((always_inline)) {
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
                pa_barrier();
            };
            auto request_next = [&]() __attribute__((always_inline)) {
                if (k_tile < t_end) request_keys(PHASED ? s2 : s0);
                if (v_tile < t_end) request_values(s1);
            };
            auto turn = [&]() __attribute__((always_inline)) {
                const int s = s0;
                s0 = s1, s1 = PHASED ? s2 : s, s2 = s;
            };
            // tiles that this wave's rows see end here; in later ones it asks for its part of the tile and keeps step
            int own_end = (wave_most + PA_KEYS - 1) / PA_KEYS - skip;
            own_end = own_end < t_end ? own_end : t_end;
            request_keys(s0);
            if (p.q_whole) request_queries();
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            asm volatile("" ::: "memory");
            read_queries();
            // Scores are scaled inside the exponent.  That wants a positive scale: the sign of a negative one moves into Q^T, and a zero one
            // becomes the smallest normal number, under which scores up to 1e31 scale to the same probabilities (2^-23 apart).
            if (scale < 0.f) {
                scale = -scale;
#pragma unroll
                for (int i = 0; i < KS + RS; ++i) qf[i] = __builtin_bit_cast(frag, __builtin_bit_cast(u32x4, qf[i]) ^ 0x80008000u);
            }
            if (scale == 0.f) scale = 1.17549435e-38f;
            pa_barrier();                                      // the first tile's keys have landed, the queries are in registers
            request_values(s0);
            if (k_tile < t_end) request_keys(s1);
            if (late) pa_barrier();
            int t = t_begin;
            auto idle = [&]() __attribute__((always_inline)) {
                end_products();
                request_next();
                if (PHASED) pa_barrier();
                turn();
            };
            // (nor, where the first keys do not stay visible, those in front of its own first window)
            if (WINDOW && p.sinks == 0) {
                int own_begin = from_of(wave_least) / PA_KEYS - skip;
                own_begin = own_begin < own_end ? own_begin : own_end;
                for (; t < own_begin; ++t) idle();
            }
            if (t < own_end) {
                products(yes, no, s0, s2);
                end_products();
                request_next();
                softmax(t);
                if (PHASED) pa_barrier();
                turn();
                for (++t; t < own_end; ++t) {
                    __builtin_amdgcn_s_setprio(1);
                    products(yes, yes, s0, s2);
                    __builtin_amdgcn_s_setprio(0);
                    end_products();
                    request_next();
                    softmax(t);
                    if (PHASED) pa_barrier();
                    turn();
                }
                products(no, yes, s0, s2);
            }
            for (; t < t_end; ++t) idle();
            if (PHASED && !late) pa_barrier();                 // (as many as the other half)
        }

        // Results through LDS (each wave in memory of its own, which no wave reads any more), 256 bytes of a row at a time, so that a store writes
        // whole cache lines.
        const float total = pa_other_sum(l_run);
        const long long row_at = (long long)(q0 + tok) * (p.kv_heads * p.group) + head;
        const int rows_here = rows - (tile * ROWS + 32 * w);   // of this wave's 32
        constexpr int OP = D == 128 ? 256 : 128;               // bytes of a row of results
        const uint32_t o_lds = lds0 + w * (32 * 256);
        pa_barrier();
        if (splits > 1) {
            const long long at = row_at * p.splits + split;
#pragma unroll
            for (int part = 0; part < CT / 2; ++part) {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f32x16 &x = o[2 * part + c];
                        const f32x4 v = {x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
                        *(__attribute__((address_space(3))) f32x4 *)(o_lds + n * 256 + 16 * ((8 * c + 2 * j + half) ^ (n & 15))) = v;
                    }
                asm volatile("" ::: "memory");
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = 4 * i + l / 16, piece = l % 16;
                    const f32x4 v = lds_frag<f32x4>(o_lds + r * 256 + 16 * (piece ^ (r & 15)));
                    const long long to = of_row(at, r);
                    if (r < rows_here) *reinterpret_cast<f32x4 *>(p.part_o + to * D + 64 * part + 4 * piece) = v;
                }
                asm volatile("" ::: "memory");
            }
            if (half == 0 && n < rows_here) {
                const f32x2 ml = {m_run, total};
                *reinterpret_cast<f32x2 *>(p.part_ml + at * 2) = ml;
            }
        } else {
            // a row that sees no key is zeros
            const float inv = sees > 0 ? 1.0f / total : 0.f;
            if (p.lse && half == 0 && n < rows_here) p.lse[row_at] = sees > 0 ? (m_run + __builtin_amdgcn_logf(total)) * 0.693147180559945f : -INFINITY;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    // the halves exchange what makes eight neighbouring channels of either
                    uint32_t x[2][2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i) x[k][i] = E::pack(o[c][8 * j + 4 * k + 2 * i] * inv, o[c][8 * j + 4 * k + 2 * i + 1] * inv);
                    const auto r0 = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false), r1 = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
                    const u32x4 v = {r0[0], r1[0], r0[1], r1[1]};
                    *(__attribute__((address_space(3))) u32x4 *)(o_lds + n * OP + 16 * ((4 * c + 2 * j + half) ^ (D == 128 ? n & 15 : (n >> 1) & 7))) = v;
                }
            asm volatile("" ::: "memory");
            const long long o_at = (long long)(q0 + tok) * p.o_t + (long long)head * p.o_h;
#pragma unroll
            for (int i = 0; i < 32 * OP / 1024; ++i) {
                const int r = i * PER + l / (OP / 16), piece = l % (OP / 16);
                const u32x4 v = lds_frag<u32x4>(o_lds + r * OP + 16 * (piece ^ (D == 128 ? r & 15 : (r >> 1) & 7)));
                const long long to = of_row(o_at, r);
                if (r < rows_here) *reinterpret_cast<u32x4_a2 *>(p.out + to + 8 * piece) = v;
            }
        }
        if (slot + (int)(gridDim.x >> 3) < here) {
            pa_barrier();                                      // (its requests write over the results)
            c = scan(0);
        }
    }
}

// The pieces of split rows.  out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.  A wave takes `each` rows, one after the other; of
// a row, a lane works out the weight of a piece, then eight pieces' outputs are on their way at a time.  Rows of a sequence whose keys were
// not divided are stepped over together (54000 rows of 2 such sequences: 3 us; with a wave to a row, each looking its sequence up, 9).
template <typename E, int D>
__global__ __launch_bounds__(256, 8) void prompt_merge_kernel(const PaParams p, const int each)
{
    constexpr int LANES = D / 4, AT_ONCE = 64 / LANES;     // lanes to a piece, four channels each; pieces to a load
    const int l = threadIdx.x & 63;
    const int heads = p.kv_heads * p.group;
    const long long first = ((long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * each, all = p.total_q * heads;
    const long long end = first + each < all ? first + each : all;
    if (first >= end) return;
    int tq = (int)(first / heads), head = (int)(first - (long long)tq * heads);
    int b = __builtin_amdgcn_readfirstlane(sequence_of(p.cu_q, p.B, tq));
    for (long long r = first; b < p.B; ++b) {
        const Span sq = span_of(p.cu_q, b, (int)p.total_q), sk = span_of(p.cu_k, b, (int)p.total_k);
        const int splits = pa_splits_of(pa_tiles_of(sk.len, p.most_tiles), p.split_tiles, p.splits);
        if (tq < sq.begin) tq = sq.begin, head = 0, r = (long long)tq * heads;
        if (r >= end) return;
        if (splits <= 1) {                                 // written by the attention kernel
            if (tq < sq.begin + sq.len) tq = sq.begin + sq.len, head = 0, r = (long long)tq * heads;
            continue;
        }
        for (; r < end && tq < sq.begin + sq.len; ++r, tq += head + 1 == heads, head = head + 1 == heads ? 0 : head + 1) {
            const int sees = pa_visible(tq - sq.begin, sq.len, sk.len, p.causal);
            const f32x2 *const ml = reinterpret_cast<const f32x2 *>(p.part_ml) + r * p.splits;
            const int part = l / LANES, ch = 4 * (l % LANES);
            const float *po = p.part_o + r * p.splits * D;
            f32x4 x[4];
            auto load = [&](const int i0) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = i0 + j * AT_ONCE + part;
                    x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if (i < splits) x[j] = *reinterpret_cast<const f32x4 *>(po + (uint32_t)(i * D + ch));
                }
            };
            f32x2 mine[PA_MAX_SPLITS / 64];
            float top = PA_LOW;
#pragma unroll
            for (int i = 0; i < PA_MAX_SPLITS / 64; ++i) {
                mine[i] = f32x2{PA_LOW, 0.f};
                if (64 * i + l < splits) mine[i] = ml[64 * i + l];
                top = fmaxf(top, mine[i][0]);
            }
            load(0);
#pragma unroll
            for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
            float total = 0.f, weight[PA_MAX_SPLITS / 64];
#pragma unroll
            for (int i = 0; i < PA_MAX_SPLITS / 64; ++i) {
                weight[i] = __builtin_amdgcn_exp2f(mine[i][0] - top);
                total += weight[i] * mine[i][1];
            }
#pragma unroll
            for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);

            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int i0 = 0; i0 < splits; i0 += 4 * AT_ONCE) {
                if (i0 > 0) load(i0);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = i0 + j * AT_ONCE + part;         // (of the same 64 for all lanes)
                    const float a = __shfl(i0 < 64 ? weight[0] : weight[PA_MAX_SPLITS / 64 - 1], i & 63);
                    if (i < splits) acc += a * x[j];
                }
            }
#pragma unroll
            for (int d = LANES; d < 64; d *= 2)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += __shfl_xor(acc[j], d);
            const float inv = sees > 0 ? 1.0f / total : 0.f;
            if (part == 0) {
                uint16_t *dst = p.out + (long long)tq * p.o_t + (long long)head * p.o_h + ch;
                *reinterpret_cast<u32x2_a2 *>(dst) = u32x2{E::pack(acc[0] * inv, acc[1] * inv), E::pack(acc[2] * inv, acc[3] * inv)};
            }
            if (p.lse && l == 0) p.lse[r] = sees > 0 ? (top + __builtin_amdgcn_logf(total)) * 0.693147180559945f : -INFINITY;
        }
    }
}

template <typename E, int D, int R, bool WINDOW>
hipError_t launch_of(const PaParams &p, hipStream_t stream)
{
    if (p.waves == 4) hipLaunchKernelGGL((prompt_attention_kernel<E, D, R, 4, WINDOW>), dim3((unsigned)p.grid), dim3(64 * 4), 0, stream, p);
    if constexpr (D == 128) {
        if (p.waves == 8) hipLaunchKernelGGL((prompt_attention_kernel<E, D, R, 8, WINDOW>), dim3((unsigned)p.grid), dim3(64 * 8), 0, stream, p);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits <= 1) return e;
    const long long rows = p.total_q * p.kv_heads * p.group, waves = 64ll * p.cus, each = (rows + waves - 1) / waves;
    hipLaunchKernelGGL((prompt_merge_kernel<E, D>), dim3((unsigned)((rows + 4 * each - 1) / (4 * each))), dim3(256), 0, stream, p, (int)each);
    return hipGetLastError();
}

template <typename E, bool WINDOW>
hipError_t launch_type(const PaParams &p, hipStream_t stream)
{
    if (p.d == 64) return launch_of<E, 64, 0, WINDOW>(p, stream);
    return p.rope ? launch_of<E, 128, PA_ROPE, WINDOW>(p, stream) : launch_of<E, 128, 0, WINDOW>(p, stream);
}

}  // namespace

hipError_t prompt_attention_launch(const PaParams &p, hipStream_t stream)
{
    if (p.window > 0) return p.fp16 ? launch_type<F16, true>(p, stream) : launch_type<BF16, true>(p, stream);
    return p.fp16 ? launch_type<F16, false>(p, stream) : launch_type<BF16, false>(p, stream);
}

}  // namespace pto
