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
#include <cmath>

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
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
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

// A sequence as the kernels take it: whatever the tables of beginnings say, inside the tensors.
struct Span {
    long long begin;
    int len;
};
__device__ __forceinline__ Span span_of(const int32_t *cu, const int b, const long long total)
{
    long long lo = cu[b], hi = cu[b + 1];
    lo = lo < 0 ? 0 : (lo > total ? total : lo);
    hi = hi < lo ? lo : (hi > total ? total : hi);
    return {lo, (int)(hi - lo)};
}

// Keys that local token t of a sequence sees.
__device__ __forceinline__ int pa_visible(const int t, const int lq, const int lk, const int causal)
{
    if (!causal) return lk;
    const int n = t + 1 + lk - lq;
    return n < 0 ? 0 : (n > lk ? lk : n);
}

// 16-byte pieces of a tile in LDS: piece c of row r lies at c ^ swizzle(r), so that neither 16 lanes that read one piece of 16
// key rows nor 16 lanes that read four rows' 32 value channels meet in a bank.  DMA writes pieces in order, so the permutation is in
// what each lane asks for.
__device__ __forceinline__ int pa_swizzle_k128(const int r) { return r & 15; }
__device__ __forceinline__ int pa_swizzle_k64(const int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int pa_swizzle_v128(const int r) { return 4 * (r & 3); }
__device__ __forceinline__ int pa_swizzle_v64(const int r) { return 4 * ((r >> 1) & 1); }

template <typename E, int D, int R, int W>
__global__ __launch_bounds__(64 * W, 2) void prompt_attention_kernel(const PaParams p)
{
    constexpr int ROWS = 32 * W;
    constexpr int KP = D * 2;                              // bytes of a key row, and of a value row
    constexpr int K_BYTES = PA_KEYS * KP, R_BYTES = PA_KEYS * R * 2;
    constexpr int STAGE = 2 * K_BYTES + R_BYTES;           // [keys | rope keys | values]
    constexpr int KS = D / 16, RS = R / 16, CT = D / 32;
    constexpr int NK = K_BYTES / 1024 / W, NR = R_BYTES / 1024 / W;   // requests of a wave per tile: keys (as many values), rope keys
    static_assert(K_BYTES % (1024 * W) == 0 && R_BYTES % (1024 * W) == 0, "whole requests for every wave");
    typedef typename E::frag frag;

    __shared__ __attribute__((aligned(1024))) uint8_t pool[2 * STAGE];

    const int tid = threadIdx.x, l = tid & 63, n = l & 31, half = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    // Workgroup -> (key head, sequence, row tile, split).  An XCD takes consecutive items, so that workgroups which read the same
    // head's keys share an L2; a sequence's last rows, which see the most keys, come first.
    const long long per_xcd = (p.items * p.kv_heads + 7) / 8;
    const long long item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (item >= p.items * p.kv_heads || (blockIdx.x >> 3) >= per_xcd) return;
    const int kvh = (int)(item / p.items);
    long long rest = item - kvh * p.items;
    int b = -1, lq = 0, lk = 0, tiles = 0, splits = 1;
    long long q0 = 0, k0 = 0;
    for (int base = 0; base < p.B; base += 64) {
        const int mine = base + l;
        Span sq = {0, 0}, sk = {0, 0};
        int mt = 0, ms = 1;
        if (mine < p.B) {
            sq = span_of(p.cu_q, mine, p.total_q);
            sk = span_of(p.cu_k, mine, p.total_k);
            mt = (int)(((long long)sq.len * p.group + ROWS - 1) / ROWS);
            ms = pa_splits_of((sk.len + PA_KEYS - 1) / PA_KEYS, p.split_tiles, p.splits);
        }
        long long upto = (long long)mt * ms;               // items of this and all sequences before it (of these 64)
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const long long o = __shfl_up(upto, d);
            upto += l >= d ? o : 0;
        }
        const uint64_t past = __ballot(upto > rest);
        if (past != 0) {
            const int who = __builtin_ctzll(past);
            b = base + who;
            rest -= who > 0 ? __shfl(upto, who - 1) : 0;
            lq = __shfl(sq.len, who), lk = __shfl(sk.len, who);
            q0 = __shfl(sq.begin, who), k0 = __shfl(sk.begin, who);
            tiles = __shfl(mt, who), splits = __shfl(ms, who);
            break;
        }
        rest -= __shfl(upto, 63);
    }
    if (b < 0) return;
    lq = __builtin_amdgcn_readfirstlane(lq), lk = __builtin_amdgcn_readfirstlane(lk), splits = __builtin_amdgcn_readfirstlane(splits);
    const int which = __builtin_amdgcn_readfirstlane((int)(rest / splits));
    const int split = __builtin_amdgcn_readfirstlane((int)rest - which * splits);
    const int tile = p.causal ? __builtin_amdgcn_readfirstlane(tiles) - 1 - which : which;

    // This lane's row, and how many keys it sees.  Rows past the last one stand in with it and are never stored.
    const int rows = lq * p.group;
    const int row = tile * ROWS + 32 * w + n;
    const int row_in = row < rows ? row : rows - 1;
    const int tok = row_in / p.group, head = kvh * p.group + row_in - tok * p.group;
    const int sees = pa_visible(tok, lq, lk, p.causal);
    const int last_row = tile * ROWS + ROWS - 1 < rows ? tile * ROWS + ROWS - 1 : rows - 1;
    const int wg_sees = pa_visible(last_row / p.group, lq, lk, p.causal);
    const int wave_most = tile * ROWS + 32 * w < rows ? pa_visible(__builtin_amdgcn_readlane(tok, 31), lq, lk, p.causal) : 0;
    const int wave_least = pa_visible(__builtin_amdgcn_readlane(tok, 0), lq, lk, p.causal);

    const int key_tiles = (wg_sees + PA_KEYS - 1) / PA_KEYS;
    const int split_len = (key_tiles + splits - 1) / splits;
    const int t_begin = split * split_len;
    const int t_end = t_begin + split_len < key_tiles ? t_begin + split_len : key_tiles;

    frag qf[KS + RS];
    {
        const uint16_t *qrow = p.q + (q0 + tok) * p.q_t + head * p.q_h + 8 * half;
#pragma unroll
        for (int i = 0; i < KS; ++i) qf[i] = __builtin_bit_cast(frag, (u32x4) * reinterpret_cast<const u32x4_a2 *>(qrow + 16 * i));
        if (R > 0) {
            const uint16_t *rrow = p.qr + (q0 + tok) * p.qr_t + head * p.qr_h + 8 * half;
#pragma unroll
            for (int i = 0; i < RS; ++i) qf[KS + i] = __builtin_bit_cast(frag, (u32x4) * reinterpret_cast<const u32x4_a2 *>(rrow + 16 * i));
        }
    }
    // Scores are scaled inside the exponent.  That wants a positive scale: the sign of a negative one moves into Q^T, and a zero one
    // becomes the smallest normal number, under which every finite score scales to the same probabilities.
    float scale = p.scale_log2;
    if (scale < 0.f) {
        scale = -scale;
#pragma unroll
        for (int i = 0; i < KS + RS; ++i) qf[i] = __builtin_bit_cast(frag, __builtin_bit_cast(u32x4, qf[i]) ^ 0x80008000u);
    }
    if (scale == 0.f) scale = 1.17549435e-38f;

    // Requests of a tile: a wave's request brings 1024 bytes of whole rows.  Keys past the sequence's last one stand in with it (their
    // probabilities are zero, and what lies behind the sequence is never touched).
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte_t *)pool;
    const uint8_t *const k_base = reinterpret_cast<const uint8_t *>(p.k + k0 * p.k_t + kvh * p.k_h);
    const uint8_t *const v_base = reinterpret_cast<const uint8_t *>(p.v + k0 * p.v_t + kvh * p.v_h);
    const uint8_t *const r_base = R > 0 ? reinterpret_cast<const uint8_t *>(p.kr + k0 * p.kr_t + kvh * p.kr_h) : nullptr;
    constexpr int PER = 1024 / KP;                         // rows of a request
    const int krow = l / (KP / 16), kpiece = l % (KP / 16);
    const int rrow = l / 8, rpiece = l % 8;
    auto request = [&](const int t, const int stage) __attribute__((always_inline)) {
        const int left = lk - t * PA_KEYS;
        const uint8_t *kb = k_base + (long long)t * PA_KEYS * p.k_t * 2, *vb = v_base + (long long)t * PA_KEYS * p.v_t * 2;
        const uint32_t dst = lds0 + stage * STAGE;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int req = i * W + w, r = req * PER + krow;
            const int from = r < left ? r : left - 1;
            const int ck = kpiece ^ (D == 128 ? pa_swizzle_k128(r) : pa_swizzle_k64(r)), cv = kpiece ^ (D == 128 ? pa_swizzle_v128(r) : pa_swizzle_v64(r));
            dma16_base(kb, (uint32_t)from * (uint32_t)(p.k_t * 2) + 16 * ck, dst + req * 1024);
            dma16_base(vb, (uint32_t)from * (uint32_t)(p.v_t * 2) + 16 * cv, dst + K_BYTES + R_BYTES + req * 1024);
        }
        if (R > 0) {
            const uint8_t *rb = r_base + (long long)t * PA_KEYS * p.kr_t * 2;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int req = i * W + w, r = req * 8 + rrow;
                const int from = r < left ? r : left - 1;
                dma16_base(rb, (uint32_t)from * (uint32_t)(p.kr_t * 2) + 16 * (rpiece ^ pa_swizzle_k64(r)), dst + K_BYTES + req * 1024);
            }
        }
    };
    constexpr int REQUESTS = 2 * NK + NR;

    f32x16 o[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
    float m_run = PA_LOW, l_run = 0.f;                     // the row's reference maximum (log2), this lane's share of its sum

    // LDS addresses of the operand reads: key row n, pieces 2 * ks + half; values: keys 4 * half + (l % 16) / 4 (+ 8), channels
    // 16 * ((l / 16) & 1) + 4 * (l % 4)
    const int ksw = (D == 128 ? pa_swizzle_k128(n) : pa_swizzle_k64(n)) ^ half, rsw = pa_swizzle_k64(n) ^ half;
    const int vkey = 4 * half + ((l & 15) >> 2);
    const int vsw = D == 128 ? pa_swizzle_v128(vkey) : pa_swizzle_v64(vkey);
    const int vlow = 2 * ((l >> 4) & 1) + ((l & 3) >> 1);

    if (t_begin < t_end) request(t_begin, 0);
    for (int t = t_begin; t < t_end; ++t) {
        const int stage = (t - t_begin) & 1;
        if (t + 1 < t_end) {
            request(t + 1, stage ^ 1);
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(REQUESTS));
        } else {
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        }
        pa_barrier();                                      // every wave's part of tile t has landed
        if (t * PA_KEYS < wave_most) {                     // (of a tile that a wave's rows do not see the wave does nothing)
            const uint8_t *kt = pool + stage * STAGE, *rt = kt + K_BYTES, *vt = rt + R_BYTES;
            f32x16 s[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[h][i] = 0.f;
#pragma unroll
                for (int i = 0; i < KS; ++i) s[h] = E::mfma(*reinterpret_cast<const frag *>(kt + (32 * h + n) * KP + 16 * ((2 * i) ^ ksw)), qf[i], s[h]);
#pragma unroll
                for (int i = 0; i < RS; ++i) s[h] = E::mfma(*reinterpret_cast<const frag *>(rt + (32 * h + n) * (R * 2) + 16 * ((2 * i) ^ rsw)), qf[KS + i], s[h]);
            }
            if ((t + 1) * PA_KEYS > wave_least) {
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
            if (__any(mx > m_run + PA_TAU)) {              // rare: the reference follows the true maximum lazily
                const float m_new = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[c][i] *= alpha;
            }
            frag pf[4];
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][8 * g + i], scale, -m_run));
                        sum += e[i];
                    }
                    const u32x4 pk = {E::pack(e[0], e[1]), E::pack(e[2], e[3]), E::pack(e[4], e[5]), E::pack(e[6], e[7])};
                    pf[2 * h + g] = __builtin_bit_cast(frag, pk);
                }
            l_run += sum;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const uint8_t *at = vt + (16 * ks + vkey) * KP + 16 * ((4 * c + vlow) ^ vsw) + 8 * (l & 1);
                    const s16x4 lo = lds_read_tr16(reinterpret_cast<const uint16_t *>(at)), hi = lds_read_tr16(reinterpret_cast<const uint16_t *>(at + 8 * KP));
                    o[c] = E::mfma(__builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), pf[ks], o[c]);
                }
        }
        pa_barrier();                                      // tile t's buffer may be written again
    }

    const float total = pa_other_sum(l_run);
    if (row >= rows) return;
    if (splits > 1) {
        const long long at = ((q0 + tok) * p.kv_heads * p.group + head) * p.splits + split;
        float *po = p.part_o + at * D;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 x = {o[c][4 * j], o[c][4 * j + 1], o[c][4 * j + 2], o[c][4 * j + 3]};
                *reinterpret_cast<f32x4 *>(po + 32 * c + 8 * j + 4 * half) = x;
            }
        if (half == 0) {
            const f32x2 ml = {m_run, total};
            *reinterpret_cast<f32x2 *>(p.part_ml + at * 2) = ml;
        }
        return;
    }
    // a row that sees no key is zeros
    const float inv = sees > 0 ? 1.0f / total : 0.f;
    uint16_t *orow = p.out + (q0 + tok) * p.o_t + head * p.o_h + 8 * half;
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
            *reinterpret_cast<u32x4_a2 *>(orow + 32 * c + 16 * j) = v;
        }
    if (p.lse && half == 0)
        p.lse[(q0 + tok) * p.kv_heads * p.group + head] = sees > 0 ? (m_run + __builtin_amdgcn_logf(total)) * 0.693147180559945f : -INFINITY;
}

// The pieces of split rows: a wave per row.  out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.
template <typename E, int D>
__global__ __launch_bounds__(256) void prompt_merge_kernel(const PaParams p)
{
    constexpr int PER = D / 64;
    const int l = threadIdx.x & 63;
    const int heads = p.kv_heads * p.group;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= p.total_q * heads) return;
    const long long tq = r / heads;
    const int head = (int)(r - tq * heads);
    const int b = sequence_of(p.cu_q, p.B, tq);
    if (b >= p.B) return;
    const Span sq = span_of(p.cu_q, b, p.total_q), sk = span_of(p.cu_k, b, p.total_k);
    if (tq < sq.begin || tq >= sq.begin + sq.len) return;
    const int splits = pa_splits_of((sk.len + PA_KEYS - 1) / PA_KEYS, p.split_tiles, p.splits);
    if (splits <= 1) return;                               // written by the attention kernel
    const int sees = pa_visible((int)(tq - sq.begin), sq.len, sk.len, p.causal);
    float top = PA_LOW;
    for (int i = l; i < splits; i += 64) top = fmaxf(top, p.part_ml[(r * p.splits + i) * 2]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    float acc[PER], total = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    for (int i = 0; i < splits; ++i) {
        const float *ml = p.part_ml + (r * p.splits + i) * 2, *po = p.part_o + (r * p.splits + i) * D + PER * l;
        const float a = __builtin_amdgcn_exp2f(ml[0] - top);
        total += a * ml[1];
#pragma unroll
        for (int j = 0; j < PER; ++j) acc[j] += a * po[j];
    }
    const float inv = sees > 0 ? 1.0f / total : 0.f;
    uint16_t *dst = p.out + tq * p.o_t + head * p.o_h + PER * l;
    if (PER == 2) {
        const uint32_t x = E::pack(acc[0] * inv, acc[PER - 1] * inv);
        dst[0] = (uint16_t)x, dst[1] = (uint16_t)(x >> 16);
    } else {
        dst[0] = (uint16_t)E::pack(acc[0] * inv, 0.f);
    }
    if (p.lse && l == 0) p.lse[r] = sees > 0 ? (top + __builtin_amdgcn_logf(total)) * 0.693147180559945f : -INFINITY;
}

template <typename E, int D, int R>
hipError_t launch_of(const PaParams &p, hipStream_t stream)
{
    const unsigned grid = (unsigned)((p.items * p.kv_heads + 7) / 8 * 8);
    if (p.waves == 8) hipLaunchKernelGGL((prompt_attention_kernel<E, D, R, 8>), dim3(grid), dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((prompt_attention_kernel<E, D, R, 4>), dim3(grid), dim3(256), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits <= 1) return e;
    const long long rows = p.total_q * p.kv_heads * p.group;
    hipLaunchKernelGGL((prompt_merge_kernel<E, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <typename E>
hipError_t launch_type(const PaParams &p, hipStream_t stream)
{
    if (p.d == 64) return launch_of<E, 64, 0>(p, stream);
    return p.rope ? launch_of<E, 128, PA_ROPE>(p, stream) : launch_of<E, 128, 0>(p, stream);
}

}  // namespace

hipError_t prompt_attention_launch(const PaParams &p, hipStream_t stream)
{
    return p.fp16 ? launch_type<F16>(p, stream) : launch_type<BF16>(p, stream);
}

}  // namespace pto
