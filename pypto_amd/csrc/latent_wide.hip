// Attention over the cached latents for sequences of many rows, gfx950: 128 rows to a workgroup of four waves (latent_attention.hip has the
// formulas, the division of the work, and a form of 64 rows for sequences of few).
//
// Per tile of 32 keys:
//   scores: wave w multiplies all keys with rows 32w .. +31 over 576 channels (v_mfma_f32_32x32x16_bf16, Q^T in 128 registers and, its rope part, LDS): lane
//           (row, half) gets sixteen keys of its row, so a row's maximum and sum need one exchange between two lanes;
//   values: wave w owns 128 value channels of all 128 rows (all 256 accumulation registers): each transposed V operand serves four products;
//           the probabilities go round through LDS.
// While tile n's scores are made, tile n + 1 is de-quantised into LDS out of registers, and each register asks for tile n + 2 as soon as it is free; beside
// the products against V of tile n - 1 stands the softmax of tile n.  One barrier per tile, three tile buffers.
//
// Why 128 rows: a tile's 32 keys are read from LDS once by each wave for its scores, 147 KB, and eight waves with 16 rows each read as much for
// half the rows.
//
// Bound by the matrix cores and what the waves issue beside them: a tile takes 4000 clocks, of which 2176 are products (half of them scores, half values, a SIMD's one wave has both);
// scores' 36 products take some 2300 clocks with the next tile's de-quantisation and requests among them, the 32 against V some 1500 with the softmax.  Of a workgroup's whole time, ends and
// beginnings too, products take 45 %, vector instructions 38, LDS 33 and its conflicts 7, and waves wait for 25 (counters).  Trees of 25 to 63 tokens of 24 sequences,
// 128 heads, over 500 to 9000 keys: 1340 to 1410 us, 920 to 970 TFLOP/s of the products that the masks ask for; the form of 64 rows 1660.  Not kept: a tile's first
// operands read across a second barrier (1 to 2 % slower).
#include "latent_line.h"

namespace pto {
namespace {

constexpr int ROWS = LA_WIDE_ROWS, THREADS = LA_WIDE_THREADS;
constexpr int P_AT = 3 * TILE;                            // two buffers of P^T: [k-step][row group][lane] 16 bytes
constexpr int P_BYTES = 8192;
constexpr int ALPHA_AT = P_AT + 2 * P_BYTES;              // two buffers: rescale factors of the 128 rows, then which groups have one
constexpr int ALPHA_BYTES = ROWS * 4 + 16;
constexpr int Q_ROPE_AT = ROWS * DN * 2;                  // the queries come to 128 x 1024 bytes of tiles' memory, their rope parts, 128 x 128, stay here
constexpr int POOL = Q_ROPE_AT + ROWS * DR * 2;
static_assert(ALPHA_AT + 2 * ALPHA_BYTES <= Q_ROPE_AT, "the rope parts lie behind everything else");
constexpr int KSTEPS = (DN + DR) / 16;
constexpr int PIECE = ROWS * DN;

// O^T stays in the accumulation registers: anything but products on it, inside the loop, would move it into the others.
__device__ __forceinline__ void acc_product(f32x16 &acc, const bf16x8 a, const bf16x8 b) { acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0); }
// (a product of zeros: written one by one, a block's registers would come together in the others first)
// A product needs two wait states behind a vector instruction that wrote one of its operands, and for products in assembly the compiler counts none: here
// the zeros were written last, and without the wait the first block was what had been in their registers.
__device__ __forceinline__ void acc_clear(f32x16 &acc)
{
    const bf16x8 zero = {};
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(acc) : "v"(zero));
}
__device__ __forceinline__ void acc_scale(f32x16 &acc, const float alpha)
{
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float e = acc[r], tmp;
        asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %2, %1\n\ts_nop 0\n\tv_accvgpr_write_b32 %0, %1" : "+a"(e), "=&v"(tmp) : "v"(alpha));
        acc[r] = e;
    }
}
__device__ __forceinline__ f32x4 acc_read(const f32x16 &acc, const int q4)
{
    float r0, r1, r2, r3;
    asm volatile("v_accvgpr_read_b32 %0, %4\n\tv_accvgpr_read_b32 %1, %5\n\tv_accvgpr_read_b32 %2, %6\n\tv_accvgpr_read_b32 %3, %7"
                 : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
                 : "a"(acc[4 * q4]), "a"(acc[4 * q4 + 1]), "a"(acc[4 * q4 + 2]), "a"(acc[4 * q4 + 3]));
    return f32x4{r0, r1, r2, r3};
}
// The scores' accumulator stays out of them: products on one destination after the other (no wait states among them), then the wait
// that a vector instruction's read needs.  Their operands come from LDS, or stay in registers from before the loop (a wait in front of each cost 1 %):
// whether the compiler put a copy in front of one anyway is read from its listing by tests/test_product_waits.py.
__device__ __forceinline__ void s_product_first(f32x16 &s, const bf16x8 a, const bf16x8 b) { asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(a), "v"(b)); }
__device__ __forceinline__ void s_product(f32x16 &s, const bf16x8 a, const bf16x8 b) { asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(a), "v"(b)); }
__device__ __forceinline__ void s_done(f32x16 &s) { asm volatile("s_nop 15\n\ts_nop 3" : "+v"(s)); }
__device__ __forceinline__ void products_to_vector() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
__device__ __forceinline__ void vector_to_products() { asm volatile("s_nop 4" ::: "memory"); }

// EIGHTS: pages and the cache hold whole eights of rows.
template <bool EIGHTS>
__global__ __launch_bounds__(THREADS) void latent_attention_wide_kernel(const LaParams p)
{
    __shared__ __attribute__((aligned(16))) uint8_t pool[POOL];

    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t pool_lds = (uint32_t)(uintptr_t)(lds_byte_t *)pool;

    __shared__ LineTable<THREADS> table;
    if (p.form && constant(p.form) == 0) return;           // (the other form had the call)
    const Line<ROWS, THREADS, false> line(p, table);
    if (!line.begin()) return;
    Place at;
    int i_begin, i_end;
    while (line.next(at, i_begin, i_end)) {
        const int l = (int)opaque(tid & 63), half = l >> 5, col = l & 31;
        const Sight<ROWS> sight(p, at);
        const int last = sight.last;                       // of the row tile's rows
        i_end = i_end < sight.tiles ? i_end : sight.tiles;
        const int ntiles = i_end > i_begin ? i_end - i_begin : 0;
        auto key_of_tile = [&](const int n) { return sight.first_key(i_begin + n); };
        f32x16 o[16];                                      // block 4*rg + c: rows 32*rg .., value channels at 128w + 32c ..
#pragma unroll
        for (int i = 0; i < 16; ++i) acc_clear(o[i]);
        float m_run = LOW, l_run = 0.f;                    // of this lane's row: reference maximum, log2 domain; sum of exp2(s - m_run)

        if (ntiles > 0) {                                  // uniform
            // Gather: wave w takes keys 8w .. 8w+7 of every tile, eight lanes each, a lane 64 channels of the latents (one scale) and eight of the
            // rope part.
            u32x4 raw[4], raw_rope;
            float raw_scale, next_scale;
            constexpr int NEAR = EIGHTS ? 8 : 1;
            auto row_of_tile = [&](const int n) __attribute__((always_inline)) { return page_of<NEAR>(p, at, key_of_tile(n) + 8 * w + (EIGHTS ? 0 : l >> 3)); };
            Page page = row_of_tile(0), page1 = row_of_tile(1), page2 = row_of_tile(2);
            // (what hangs on the lane alone is made where it is used: kept, it would take the registers of the products' operands)
            auto lane = [&]() {
                uint32_t x = tid & 63;
                asm volatile("" : "+v"(x));
                return x;
            };
            auto ask_latent = [&](const RowAt &row, const int i) __attribute__((always_inline)) {
                const uint32_t x = lane();
                raw[i] = global<u32x4>(row.nope + 16 * i, (EIGHTS ? x >> 3 : 0) * (uint32_t)p.cache.nope_pitch + 64 * (x & 7));
            };
            auto ask_scale = [&](const RowAt &row) __attribute__((always_inline)) {
                const uint32_t x = lane();
                next_scale = global<float>(row.scale, (EIGHTS ? x >> 3 : 0) * (uint32_t)p.cache.scale_pitch + 4 * ((x & 7) >> 1));
            };
            auto ask_rope = [&](const RowAt &row) __attribute__((always_inline)) {
                const uint32_t x = lane();
                raw_rope = global<u32x4>(row.rope, (EIGHTS ? x >> 3 : 0) * (uint32_t)p.cache.rope_pitch + 16 * (x & 7));
            };
            // A tile's rows into LDS, in 32 pieces of two values per lane (one to a product: five vector instructions fit beside it) and one of the rope
            // channels.  Of a row's 64 latent pieces of eight channels number 4 j + k lies at k * 16 + j.
            const uint32_t emit_off = (uint32_t)((8 * w + (l >> 3)) * PITCH + 32 * (l & 7));
            u32x4 dq;
            auto emit = [&](const uint32_t tile, const int d) __attribute__((always_inline)) {
                const uint32_t r = raw[d >> 3][(d >> 1) & 3];
                dq[d & 3] = d & 1 ? dequant_upper(r, raw_scale) : dequant_lower(r, raw_scale);
                if ((d & 3) == 3) *reinterpret_cast<u32x4 *>(pool + tile + emit_off + 256 * ((d >> 2) & 3) + 16 * (d >> 4)) = dq;
            };
            auto emit_rope = [&](const uint32_t tile) __attribute__((always_inline)) {
                *reinterpret_cast<u32x4 *>(pool + tile + emit_off + (DN * 2 - 16 * (lane() & 7))) = raw_rope;
            };
            // Queries: a wave's own 32 rows, a row's latent part per request, 16-byte chunk i of row j at i ^ (j & 15).  Rows past the last one
            // read it and are never stored.
            const uint32_t q_lds = pool_lds + w * (32 * DN * 2);
#pragma unroll 4
            for (int j = 0; j < 32; ++j) {
                const int r = sight.row0 + (32 * w + j < last ? 32 * w + j : last);
                const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                dma16_base(p.q + (long long)(at.q0 + tok) * p.q_t + (long long)head * p.q_h, (uint32_t)(16 * (l ^ (j & 15))), q_lds + j * (DN * 2));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 8 * i + (l >> 3), r = sight.row0 + (32 * w + j < last ? 32 * w + j : last);
                const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                dma16(p.qr + (long long)(at.q0 + tok) * p.qr_t + (long long)head * p.qr_h + 8 * ((l & 7) ^ (j & 7)), pool_lds + Q_ROPE_AT + (4 * w + i) * 1024);
            }

            {
                const RowAt row = row_at(p, page);
                ask_scale(row);
                ask_rope(row);
#pragma unroll
                for (int i = 0; i < 4; ++i) ask_latent(row, i);
            }
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));      // (the queries too)
            asm volatile("" ::: "memory");
            bf16x8 qf[DN / 16];                            // Q^T: lane (row, half) holds channels 16*ks + 8*half .. +7
#pragma unroll
            for (int ks = 0; ks < DN / 16; ++ks) qf[ks] = *reinterpret_cast<const bf16x8 *>(pool + (32 * w + col) * (DN * 2) + 16 * ((2 * ks + half) ^ (col & 15)));
            float sc_log2 = p.scale_log2;                  // (its sign moves into Q^T, zero becomes the smallest normal number)
            if (sc_log2 < 0.f) {
                sc_log2 = -sc_log2;
#pragma unroll
                for (int i = 0; i < DN / 16; ++i) qf[i] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, qf[i]) ^ 0x80008000u);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u32x4 *const at_rope = reinterpret_cast<u32x4 *>(pool + Q_ROPE_AT + (4 * w + i) * 1024 + 16 * l);
                    *at_rope = *at_rope ^ 0x80008000u;
                }
            }
            if (sc_log2 == 0.f) sc_log2 = 1.17549435e-38f;
            __syncthreads();                               // every wave has its queries: the tiles may go over them
            raw_scale = next_scale;
            check_scale<8>(raw_scale, raw_rope);
            {                                              // (in the order of the loop's requests, or its first waits would be for the wrong ones)
                const RowAt row = row_at(p, page1);
                ask_scale(row);
                emit_rope(0);
                ask_rope(row);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int d = 0; d < 8; ++d) emit(0, 8 * i + d);
                    ask_latent(row, i);
                }
            }

            const int krow = tile_row_of(col);
            const uint32_t kbase = (uint32_t)(krow * PITCH + 256 * half), rbase = (uint32_t)(krow * PITCH + DN * 2 + 16 * half);
            const uint32_t vbase = (uint32_t)((half + 4 * ((l & 15) >> 2)) * PITCH + 32 * ((l >> 4) & 1) + 8 * (l & 3) + 256 * w);
            f32x16 s;
            u32x4 pk0, pk1;
            float mx = 0.f, m_new = 0.f, alpha = 1.f, lsum = 0.f;
            bool upd = false;
            bf16x8 vf[3], pf[4];                           // V^T of product block (kk, c) in vf[(4 * kk + c) % 3]
            uint32_t seen = ~0u;                           // of the tile in s: the keys that this lane's row sees
            bool cut = false;                              // some row does not see them all
            auto load_v = [&](const uint32_t tile, const int i) __attribute__((always_inline)) {
                const uint16_t *a0 = reinterpret_cast<const uint16_t *>(pool + tile + vbase + 16 * (i >> 2) * PITCH + 64 * (i & 3));
                const s16x4 lo = lds_read_tr16(a0), hi = lds_read_tr16(a0 + PITCH);            // (two rows on)
                vf[i % 3] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            auto load_p = [&](const int pbuf, const int kk, const int rg) __attribute__((always_inline)) {
                pf[rg] = *reinterpret_cast<const bf16x8 *>(pool + P_AT + pbuf * P_BYTES + ((kk * 4 + rg) * 64 + l) * 16);
            };
            auto look = [&](const int n) __attribute__((always_inline)) {
                const uint32_t first = key_of_tile(n);
                cut = !sight.whole(first);                 // (uniform)
                if (cut) {
                    const int row = sight.row0 + 32 * w + (int)(lane() & 31), tok = divide(row < sight.rows ? row : sight.rows - 1, p.of_heads);
                    // (bit tile_row_of(i + 4) is one above bit tile_row_of(i): the upper half's keys come to the lower one's bits)
                    seen = sight.seen(first, sight.sees(tok), p.mask ? p.mask + (long long)(at.q0 + tok) * p.words : nullptr) >> (lane() >> 5);
                }
            };
            // The score products' key operands, AHEAD of their use; the rope part first, whose queries are read beside it.
            constexpr int AHEAD = 4;
            bf16x8 fa[8];
            auto read_k = [&](const uint32_t tile, const int m) __attribute__((always_inline)) {
                const int ks = m - DR / 16;
                return *reinterpret_cast<const bf16x8 *>(pool + tile + (m < DR / 16 ? rbase + 32 * m : kbase + 512 * (ks & 1) + 16 * (ks >> 1)));
            };
            // Scores of tile n, at `cur`; the next tile goes into `next`, the one behind it is asked for, and the first operands of the products
            // against V of the tile at `prev` are read.
            auto scores = [&](const uint32_t cur, const uint32_t prev, const uint32_t next, const RowAt &row, const int pbuf) __attribute__((always_inline)) {
                bf16x8 qr[DR / 16];
#pragma unroll
                for (int m = 0; m < AHEAD; ++m) fa[m] = read_k(cur, m);
#pragma unroll
                for (int e = 0; e < DR / 16; ++e) qr[e] = *reinterpret_cast<const bf16x8 *>(pool + Q_ROPE_AT + 4096 * w + 128 * (lane() & 31) + 16 * ((2 * e + half) ^ (lane() & 7)));
#pragma unroll
                for (int m = 0; m < KSTEPS; ++m) {
                    if (m == 0) s_product_first(s, fa[0], qr[0]);
                    else s_product(s, fa[m & 7], m < DR / 16 ? qr[m % (DR / 16)] : qf[m >= DR / 16 ? m - DR / 16 : 0]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (m + AHEAD < KSTEPS) fa[(m + AHEAD) & 7] = read_k(cur, m + AHEAD);
                    if (m == 1) raw_scale = next_scale, check_scale<8>(raw_scale, raw_rope);
                    if (m == 2) ask_scale(row);
                    if (m >= 3 && m < 35) emit(next, m - 3);
                    if (m >= 11 && (m - 11) % 8 == 0) ask_latent(row, (m - 11) / 8);
                    if (m == 4) emit_rope(next);
                    if (m == 5) ask_rope(row);
                    if (m >= 25 && m < 33 && (m & 1)) load_p(pbuf, 0, (m - 25) >> 1);
                    if (m == 33 || m == 34) load_v(prev, m - 33);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // The softmax of the scores in s, of tile n, in steps beside products; it leaves this wave's P^T in buffer `pbuf` and, where a running maximum
            // moved past the threshold, the rows' rescale factors beside it.
            auto softmax_step = [&](const int q, const int n, const int pbuf) __attribute__((always_inline)) {
                if (q == 0) {
                    s_done(s);
                    if (cut) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = (seen >> tile_row_of(8 * (r >> 2) + (r & 3))) & 1 ? s[r] : -INFINITY;
                    }
                    mx = fmaxf(s[0], s[1]);
                } else if (q < 4) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) mx = fmaxf(mx, fmaxf(s[4 * q - 2 + 2 * e], s[4 * q - 1 + 2 * e]));
                } else if (q == 4) {
                    mx = fmaxf(mx, fmaxf(s[14], s[15]));
                } else if (q == 5) {
                    float lo, hi;
                    both_halves(mx, lo, hi);
                    mx = fmaxf(lo, hi) * sc_log2;
                } else if (q == 6) {
                    upd = mx > m_run + TAU;
                    m_new = upd ? mx : m_run;
                    alpha = upd ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
                    m_run = m_new;
                    lsum = 0.f;
                } else if (q < 23) {                       // one exponential per product
                    const int r = q - 7;
                    s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sc_log2, -m_new));
                    lsum += s[r];
                    if (r & 1) {
                        if (r < 8) pk0[r >> 1] = pack_bf16x2(s[r - 1], s[r]);
                        else pk1[(r - 8) >> 1] = pack_bf16x2(s[r - 1], s[r]);
                    }
                } else if (q == 23) {
                    *reinterpret_cast<u32x4 *>(pool + P_AT + pbuf * P_BYTES + (w * 64 + l) * 16) = pk0;
                } else if (q == 24) {
                    *reinterpret_cast<u32x4 *>(pool + P_AT + pbuf * P_BYTES + ((4 + w) * 64 + l) * 16) = pk1;
                } else if (q == 25) {
                    float lo, hi;
                    both_halves(lsum, lo, hi);
                    l_run = l_run * alpha + (lo + hi);
                } else if (q == 26) {
                    const bool any = n > 0 && __any(upd);                                      // wave-uniform (before the first tile there is nothing to rescale)
                    uint8_t *const a = pool + ALPHA_AT + pbuf * ALPHA_BYTES;
                    if (any) reinterpret_cast<float *>(a)[32 * w + (lane() & 31)] = alpha;
                    reinterpret_cast<int *>(a + ROWS * 4)[w] = any ? 1 : 0;
                }
            };
            // O^T += V^T . P^T of the tile at `prev` (its P^T and factors in buffer pbuf), whose first operands are read; SM: with the softmax of
            // tile n beside it
            auto values = [&](auto sm_tag, const uint32_t prev, const int pbuf, const int n) __attribute__((always_inline)) {
                constexpr bool SM = decltype(sm_tag)::value;
                const i32x4 fl = *reinterpret_cast<const i32x4 *>(pool + ALPHA_AT + pbuf * ALPHA_BYTES + ROWS * 4);
                const int any = __builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]);
                if (__builtin_expect(any, 0)) {            // rare
                    products_to_vector();
#pragma unroll
                    for (int rg = 0; rg < 4; ++rg) {
                        if (__builtin_amdgcn_readfirstlane(fl[rg]) == 0) continue;
                        const float a = reinterpret_cast<const float *>(pool + ALPHA_AT + pbuf * ALPHA_BYTES)[32 * rg + col];
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc_scale(o[4 * rg + c], a);
                    }
                    vector_to_products();
                }
#pragma unroll
                for (int mp = 0; mp < 32; ++mp) {
                    const int i = mp >> 2, rg = mp & 3;    // product block i = 4 * kk + c
                    acc_product(o[4 * rg + (i & 3)], vf[i % 3], pf[rg]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (rg == 0 && i + 2 < 8) load_v(prev, i + 2);
                    if (i == 3) load_p(pbuf, 1, rg);
                    if (SM && mp > 0) softmax_step(mp - 1, n, pbuf ^ 1);
                    if (SM && mp == 28) page = row_of_tile(n + 3);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // The first turn's products against V are of the first tile itself with probabilities of zero: a turn of its own, without them, would leave
            // registers to be restored in front of the others.
            *reinterpret_cast<u32x4 *>(pool + P_AT + P_BYTES + 32 * tid) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4 *>(pool + P_AT + P_BYTES + 32 * tid + 16) = u32x4{0, 0, 0, 0};
            if (tid < 4) reinterpret_cast<int *>(pool + ALPHA_AT + ALPHA_BYTES + ROWS * 4)[tid] = 0;
            __syncthreads();
            uint32_t cur = 0, next = TILE, prev = 0;
            int pbuf = 1;                                  // of the tile at prev
            page = page2;                                  // of the tile whose rows are asked for next
            for (int n = 0; n < ntiles; ++n) {
                // (what branches stands here: around a branch among the products registers would move)
                const RowAt row = row_at(p, page);
                look(n);
                scores(cur, prev, next, row, pbuf);
                values(std::true_type{}, prev, pbuf, n);
                pbuf ^= 1;
                __syncthreads();
                const uint32_t free = n > 0 ? prev : 2 * TILE;
                prev = cur;
                cur = next;
                next = free;
            }
            // the products against V of the last tile
#pragma unroll
            for (int i = 0; i < 4; ++i) load_p(pbuf, 0, i);
            load_v(prev, 0), load_v(prev, 1);
            values(std::false_type{}, prev, pbuf, 0);
        }

        // ---- the row tile's end: see latent_attention_kernel
        products_to_vector();
        __syncthreads();
        // (what is known of the row tile comes back from LDS: see LineTable)
        const bool whole = line.one(table.whole) != 0;
        const int piece = line.one(table.piece), first = line.one(table.place.q0), rows = line.one(table.place.n) * p.heads, row0 = line.one(table.place.row_tile) * ROWS;
        float *const il = reinterpret_cast<float *>(pool + ALPHA_AT);
        if (half == 0) {
            const int r = 32 * w + col;
            if (!whole) {
                const f32x2 ml = {m_run, l_run};
                *reinterpret_cast<f32x2 *>(p.part_ml + ((long long)piece * ROWS + r) * 2) = ml;
            } else {
                il[r] = l_run == 0.f ? 0.f : 1.0f / l_run; // a row that sees no key is zeros
                if (p.lse && row0 + r < rows)
                    p.lse[(long long)first * p.heads + row0 + r] = l_run == 0.f ? -INFINITY : (m_run + __builtin_amdgcn_logf(l_run)) * 0.693147180559945f;
            }
        }
        if (!whole) {
            float *const dst = p.part_o + (long long)piece * PIECE + ((w * 64) * 64 + l) * 4;
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) *reinterpret_cast<f32x4 *>(dst + (4 * i + q4) * 256) = acc_read(o[i], q4);
        } else {
            __syncthreads();
            float iv[4];
#pragma unroll
            for (int rg = 0; rg < 4; ++rg) iv[rg] = il[32 * rg + col];
            __syncthreads();                               // (the results go over these)
#pragma unroll
            for (int rg = 0; rg < 4; ++rg)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        const f32x4 x = acc_read(o[4 * rg + c], q4) * iv[rg];
                        const u32x2 pk = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
                        const int chunk = 4 * (4 * c + q4) + w;                                  // of the row, in channel order
                        *reinterpret_cast<u32x2 *>(pool + (32 * rg + col) * (DN * 2) + 16 * (chunk ^ col) + 8 * half) = pk;
                    }
            __syncthreads();
#pragma unroll
            for (int e0 = 0; e0 < 32; e0 += 8) {
                u32x4 v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const u32x4 *>(pool + (32 * w + e0 + e) * (DN * 2) + 16 * (l ^ (e0 + e)));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = row0 + 32 * w + e0 + e;
                    if (r < rows) {
                        const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                        *reinterpret_cast<u32x4_a2 *>(p.out + (long long)(first + tok) * p.o_t + (long long)head * p.o_h + 8 * l) = v[e];
                    }
                }
            }
        }
        __syncthreads();                                   // (the next row tile's queries go over these)
    }
    line.done();
}

}  // namespace

hipError_t latent_attention_wide_launch(const LaParams &p, hipStream_t stream)
{
    if (p.bs % 8 == 0 && p.cache.rows % 8 == 0) hipLaunchKernelGGL((latent_attention_wide_kernel<true>), dim3((unsigned)p.groups), dim3(THREADS), 0, stream, p);
    else hipLaunchKernelGGL((latent_attention_wide_kernel<false>), dim3((unsigned)p.groups), dim3(THREADS), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pto
