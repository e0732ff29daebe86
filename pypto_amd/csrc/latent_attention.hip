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
// to a workgroup, so the memory for them does not depend on lengths, which the host does not know.  Where lengths decide between this form and that of 128 rows
// (latent_plan has the rule), both are launched; this one, the first, counts both's tiles, and returns if the call is the other's, or the other does.
//
// No unit is busy half of the time.  Of a workgroup's time (single tokens of 32 sequences over 2052 keys, 128 heads; counters) vector instructions take 39 %, LDS 30,
// scalar instructions 25, products 23, and its waves wait for 38 % of theirs.  A tile takes 3000 clocks (1.45 us); the selected keys' attention of 64 heads, with the same
// products and LDS traffic, 2580, at 42, 40, 10, 30 and 41 %: it has pages in LDS before its loop, where this one makes a look-up, a division and addresses for each tile, 3.3
// times as many scalar instructions in all, which is the likely difference.  Beside the tiles a beginning of 9 us (sums over the sequences 2.2, its place in the line 1.1, requests
// 1.5, their way 0.5, the first tile 3.3) and an end of 1.2, where pieces are short most of the time; and the second launch, which reads what the first wrote.
// The example 46.5 to 50 us, 17 GFLOP of products, 33 MB of pieces; 1 to 4 tokens of 90 sequences over 1016 keys, 16 heads: 42; a tree of 8 tokens over 2900 keys, 16
// heads: 22; one token with 128 heads over 30000 keys: 37.  On the way (the first of these): a look-up and a 64-bit address for each row 59, one of
// either for four neighbouring rows, pages asked for before rows, 51, boundaries moved to row tiles' edges for pieces of one tile instead of three 47.7.
#include "latent_line.h"

namespace pto {
namespace {

constexpr int P_AT = 3 * TILE;                            // two buffers of P^T: [row half][k-step][lane] 16 bytes
constexpr int P_BYTES = 4096;
constexpr int MAX_AT = P_AT + 2 * P_BYTES;                // [key half][64 rows] fp32: maxima (and at the end the sums)
constexpr int ALPHA_AT = MAX_AT + 2 * 64 * 4;             // [64 rows] fp32: rescale factors (at the end 1 / sum)
constexpr int FLAG_AT = ALPHA_AT + 64 * 4;                // two words: the last tile whose maxima moved, by parity of the tile
constexpr int POOL = FLAG_AT + 16;
constexpr int Q_ROPE_AT = LA_ROWS * DN * 2;               // query staging: 64 rows x 1024 bytes, then 64 x 128
constexpr int PIECE = LA_ROWS * DN;                       // floats of a piece's sums
constexpr int THREADS = LA_THREADS;

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

// QUADS: pages and the cache hold whole fours of rows.  CHOOSE: the form of 128 rows is launched behind this one, and p.form says whose call it is.
template <bool QUADS, bool CHOOSE>
__global__ __launch_bounds__(THREADS) void latent_attention_kernel(const LaParams p)
{
    __shared__ __attribute__((aligned(16))) uint8_t pool[POOL];

    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hq = w & 3;                                  // scores: rows 16*hq .. +15 of the workgroup's 64,
    const int kh = w >> 2;                                 // the half kh of the tile's keys
    const uint32_t pool_lds = (uint32_t)(uintptr_t)(lds_byte_t *)pool;

    __shared__ LineTable<THREADS> table;
    const Line<LA_ROWS, THREADS, CHOOSE> line(p, table);
    if (!line.begin()) return;
    Place at;
    int i_begin, i_end;
    while (line.next(at, i_begin, i_end)) {
        const int l = (int)opaque(tid & 63), half = l >> 5, col = l & 31, l16 = l & 15, quarter = l >> 4;
        const Sight<LA_ROWS> sight(p, at);
        const int last = sight.last;                       // of the row tile's rows
        i_end = i_end < sight.tiles ? i_end : sight.tiles;
        const int ntiles = i_end > i_begin ? i_end - i_begin : 0;
        auto key_of_tile = [&](const int n) { return sight.first_key(i_begin + n); };      // the first key of tile n of this piece
        // of this lane's row of scores
        const int my_row = sight.row0 + 16 * hq + l16;
        const int my_tok = divide(my_row < sight.rows ? my_row : sight.rows - 1, p.of_heads);
        const int my_sees = sight.sees(my_tok);
        const unsigned long long *const my_mask = p.mask ? p.mask + (long long)(at.q0 + my_tok) * p.words : nullptr;

        f32x16 o[4];                                       // block 2*hb + d: rows 32*hb .., value channels 64w + 32d ..
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
        float m_run = LOW;                                 // of row 16*hq + l16: reference maximum, log2 domain,
        float l_run = 0.f;                                 // and this lane's share of the sum of exp2(s - m_run)

        if (ntiles > 0) {                                  // uniform
            // Gather: wave w takes keys 4w .. 4w+3 of every tile, a quarter of its lanes each, a lane 32 channels of the latents (one scale) and
            // four of the rope part.
            struct Raw {
                u32x4 v[2];
                float sc;
                u32x2 rope;
            };
            Raw raw[2];                                    // tile n in raw[n & 1]
            constexpr int NEAR = QUADS ? 4 : 1;
            auto page_of_tile = [&](const int n) __attribute__((always_inline)) { return page_of<NEAR>(p, at, key_of_tile(n) + 4 * w + (QUADS ? 0 : quarter)); };
            Page page = page_of_tile(0), page1 = page_of_tile(1), page2 = page_of_tile(2), page3 = page_of_tile(3);
            // The queries, staged through LDS in the tile buffers 0 and 1: wave w asks for rows 8w .. 8w+7, a row's latent part per request,
            // 16-byte chunk i of row j at i ^ (j & 15) so that the fragment reads touch every bank once.  Rows past the last one read it
            // and are never stored.
            static_assert(Q_ROPE_AT + LA_ROWS * DR * 2 <= 2 * TILE, "the first tile goes to buffer 2");
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 8 * w + i, r = sight.row0 + (j < last ? j : last);
                const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                dma16_base(p.q + (long long)(at.q0 + tok) * p.q_t + (long long)head * p.q_h, (uint32_t)(16 * (l ^ (j & 15))), pool_lds + j * (DN * 2));
            }
            {
                const int j = 8 * w + (l >> 3), r = sight.row0 + (j < last ? j : last);
                const int tok = divide(r, p.of_heads), head = r - tok * p.heads;
                dma16(p.qr + (long long)(at.q0 + tok) * p.qr_t + (long long)head * p.qr_h + 8 * ((l & 7) ^ (l >> 3)), pool_lds + Q_ROPE_AT + w * 1024);
            }

            const uint32_t rows_on = QUADS ? quarter : 0;
            const uint32_t v_off = rows_on * (uint32_t)p.cache.nope_pitch + 32 * l16, sc_off = rows_on * (uint32_t)p.cache.scale_pitch + 4 * (l16 >> 2),
                           rope_off = rows_on * (uint32_t)p.cache.rope_pitch + 8 * l16;
            auto gather = [&](Raw &r, const Page k) __attribute__((always_inline)) {
                const RowAt row = row_at(p, k);
                r.v[0] = global<u32x4>(row.nope, v_off);
                r.v[1] = global<u32x4>(row.nope + 16, v_off);
                r.sc = global<float>(row.scale, sc_off);
                r.rope = global<u32x2>(row.rope, rope_off);
            };
            // The tile's rows into LDS, in eight pieces of a dword per lane and one of the rope channels.  Of a row's 64 latent pieces of eight
            // channels number 4 j + k lies at k * 16 + j: a lane's four pieces are one of each k, and lanes next to each other write next to
            // each other.
            const uint32_t emit_off = (uint32_t)((4 * w + quarter) * PITCH + 16 * l16);
            const uint32_t emit_rope_off = (uint32_t)((4 * w + quarter) * PITCH + DN * 2 + 8 * l16);
            u32x4 dq;
            auto emit = [&](Raw &r, const uint32_t tile, const int d) __attribute__((always_inline)) {
                if (d == 0) check_scale<16>(r.sc, r.rope);
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
            gather(raw[0], page);
            gather(raw[1], page1);
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));      // (the wave's queries, too)
            asm volatile("" ::: "memory");
#pragma unroll
            for (int d = 0; d < 9; ++d) emit(raw[0], 2 * TILE, d);
            gather(raw[0], page2);
            page2 = page_of_tile(4);
            if (tid < 2) reinterpret_cast<int *>(pool + FLAG_AT)[tid] = -1;
            __syncthreads();                               // the queries and the first tile are there
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
                const uint32_t first = key_of_tile(n);
                if (!sight.whole(first)) {                 // (uniform)
                    const uint32_t seen = sight.seen(first, my_sees, my_mask);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sv[e] = (seen >> key_of[e]) & 1 ? sv[e] : -INFINITY;
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
                        if (mp == 4) further = page_of_tile(n4);
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
            __syncthreads();                               // every wave has its queries: the next tile goes over them
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
        // (what is known of the row tile comes back from LDS: see LineTable)
        const bool whole = line.one(table.whole) != 0;
        const int piece = line.one(table.piece), first = line.one(table.place.q0), rows = line.one(table.place.n) * p.heads, row0 = line.one(table.place.row_tile) * LA_ROWS;
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
                p.lse[(long long)first * p.heads + row0 + r] = sum == 0.f ? -INFINITY : (m_run + __builtin_amdgcn_logf(sum)) * 0.693147180559945f;
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
                    *reinterpret_cast<u32x4_a2 *>(p.out + (long long)(first + tok) * p.o_t + (long long)head * p.o_h + 8 * l) = v[e];
                }
            }
        }
        __syncthreads();                                   // (the next row tile's queries go over these)
    }
    line.done();
}

struct JoinMemory {
    f32x4 sums[3][4][64];
    float stats[3][2][32];
};

// The pieces of row tiles that workgroups share: out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in the order of the keys.  A workgroup
// joins one accumulator block at a time (32 rows, 32 channels, as the attention kernels' registers have them) of an entry's rows, four 16-byte values to a
// lane, its four waves a quarter of the pieces each.
template <bool WIDE>
__device__ __forceinline__ void join_block(const LaParams &p, JoinMemory &mem)
{
    constexpr int TILE_ROWS = WIDE ? LA_WIDE_ROWS : LA_ROWS, BLOCKS = TILE_ROWS / 2, OF_WAVE = WIDE ? 16 : 4;
    const int block = blockIdx.x;
    if (block >= p.entries * BLOCKS) return;
    auto &sums = mem.sums;
    auto &stats = mem.stats;
    const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = l >> 5, col = l & 31;
    const int32_t *const join = p.joins + 4 * (block / BLOCKS);
    const int n = join[1];
    if (n <= 1) return;
    const int first = join[0], row0 = join[2], rows = join[3];
    const int w = (block % BLOCKS) / OF_WAVE, i = block % OF_WAVE;
    const int group = WIDE ? i >> 2 : i >> 1, c = WIDE ? i & 3 : i & 1;            // of 32 rows; of 32 of the wave's channels
    // where the pieces are: that of the first workgroup is said; the others' ranges begin inside the row tile, so it is their first
    auto place = [&](const int k) { return (long long)(k == 0 ? first : 2 * ((first >> 1) + k)); };
    float top = LOW, total = 0.f;
    f32x4 acc[4];
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) acc[q4] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto take = [&](const int k0, auto count) __attribute__((always_inline)) {
        constexpr int EACH = decltype(count)::value;       // pieces asked for at once
        f32x2 ml[EACH];
        f32x4 x[EACH][4];
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const long long at = place(k0 + 4 * j);
            ml[j] = *reinterpret_cast<const f32x2 *>(p.part_ml + (at * TILE_ROWS + 32 * group + col) * 2);
            const float *src = p.part_o + at * (TILE_ROWS * DN) + ((w * OF_WAVE + i) * 256 + l) * 4;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) x[j][q4] = *reinterpret_cast<const f32x4 *>(src + q4 * 256);
        }
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const float m = fmaxf(top, ml[j][0]), a = __builtin_amdgcn_exp2f(top - m), b = __builtin_amdgcn_exp2f(ml[j][0] - m);
            top = m;
            total = total * a + ml[j][1] * b;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) acc[q4] = acc[q4] * a + x[j][q4] * b;
        }
    };
    int k = wave;
    for (; k + 12 < n; k += 16) take(k, std::integral_constant<int, 4>{});
    for (; k < n; k += 4) take(k, std::integral_constant<int, 1>{});
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
    const int row = 32 * group + col;
    if (row >= rows) return;
    const long long r = (long long)row0 + row;
    if (p.lse && w == 0 && c == 0 && half == 0) p.lse[r] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * 0.693147180559945f;
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    const int tok = divide((int)r, p.of_heads), head = (int)r - tok * p.heads;
    uint16_t *dst = p.out + (long long)tok * p.o_t + (long long)head * p.o_h;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
        const int chunk = WIDE ? 4 * (4 * c + q4) + w : 32 * (w & 1) + 4 * (4 * c + q4) + (w >> 1);
        *reinterpret_cast<u32x2_a2 *>(dst + 8 * chunk + 4 * half) =
            u32x2{pack_bf16x2(acc[q4][0] * inv, acc[q4][1] * inv), pack_bf16x2(acc[q4][2] * inv, acc[q4][3] * inv)};
    }
}

template <bool WIDE>
__global__ __launch_bounds__(256) void latent_join_kernel(const LaParams p)
{
    __shared__ JoinMemory mem;
    join_block<WIDE>(p, mem);
}
// (five waves to a SIMD as in the other: four, with as many registers as both need, took 28 us instead of 22 for 8 trees of 30 nodes, 128 heads)
__global__ __launch_bounds__(256, 5) void latent_join_either_kernel(const LaParams narrow, const LaParams wide)
{
    __shared__ JoinMemory mem;
    if (constant(narrow.form) != 0) join_block<true>(wide, mem);
    else join_block<false>(narrow, mem);
}

}  // namespace

hipError_t latent_attention_launch(const LaParams *narrow, const LaParams *wide, hipStream_t stream)
{
    hipError_t e = hipSuccess;
    if (narrow) {
        const bool quads = narrow->bs % 4 == 0 && narrow->cache.rows % 4 == 0;
        const auto kernel = wide ? (quads ? latent_attention_kernel<true, true> : latent_attention_kernel<false, true>)
                                 : (quads ? latent_attention_kernel<true, false> : latent_attention_kernel<false, false>);
        hipLaunchKernelGGL(kernel, dim3((unsigned)narrow->groups), dim3(THREADS), 0, stream, *narrow);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (wide) {
        e = latent_attention_wide_launch(*wide, stream);
        if (e != hipSuccess) return e;
    }
    const unsigned narrow_blocks = narrow ? (unsigned)narrow->entries * (LA_ROWS / 2) : 0, wide_blocks = wide ? (unsigned)wide->entries * (LA_WIDE_ROWS / 2) : 0;
    if (!wide) hipLaunchKernelGGL((latent_join_kernel<false>), dim3(narrow_blocks), dim3(256), 0, stream, *narrow);
    else if (!narrow) hipLaunchKernelGGL((latent_join_kernel<true>), dim3(wide_blocks), dim3(256), 0, stream, *wide);
    else hipLaunchKernelGGL(latent_join_either_kernel, dim3(narrow_blocks > wide_blocks ? narrow_blocks : wide_blocks), dim3(256), 0, stream, *narrow, *wide);
    return hipGetLastError();
}

}  // namespace pto
