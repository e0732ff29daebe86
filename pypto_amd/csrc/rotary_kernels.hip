// Rotary positions, gfx950.
//
// Channel pair i of a token at position n turns by the angle n * freq[i].  The angle needs 64 bits (position 131071 in fp32
// leaves an angle 2^-7 of its bits after the point); it is reduced to the nearest quarter turn there, and what is left, at most
// pi/4, goes through the sine's and cosine's Taylor series in fp32, whose first left-out terms, x^11 / 11! and x^12 / 12!, are at most
// 1.8e-9 and 1.2e-10.  (The cosine without its tenth power is 2.5e-8 off there, 0.4 of an fp32 step.)
#include "common.h"
#include "prompt_ops.h"
#include "pypto_amd_sfa.h"

namespace pto {
namespace {

struct Turn {
    float c, s;
};

// The rounding of an angle's quotient may miss the nearest quarter turn where it is more than this, by a thousand of them at 2^63: what is
// left is then reduced again.
constexpr double TURNS_FAR = 1.0e12;

// far: set if this angle is to be asked for again, with AGAIN.
template <bool AGAIN>
__device__ __forceinline__ Turn turn_by(const double position, const double freq, const float factor, bool &far)
{
    const double angle = position * freq;
    double k = rint(angle * 0.63661977236758134308);                        // 2 / pi
    // pi / 2 as the sum of two doubles
    auto without = [](const double x, const double n) { return fma(-n, 6.123233995736766036e-17, fma(-n, 1.5707963267948965580, x)); };
    double left = without(angle, k);
    if (AGAIN) {
        const double more = rint(left * 0.63661977236758134308);
        left = without(left, more);
        k = (k - 4.0 * floor(k * 0.25)) + more;
    } else {
        far |= fabs(k) > TURNS_FAR;
    }
    const float x = (float)left, z = x * x;
    const float s = x + x * z * (-1.6666667e-1f + z * (8.3333333e-3f + z * (-1.9841270e-4f + z * 2.7557319e-6f)));
    const float c = 1.0f + z * (-0.5f + z * (4.1666667e-2f + z * (-1.3888889e-3f + z * (2.4801587e-5f + z * -2.7557319e-7f))));
    const int quarter = (int)(k - 4.0 * floor(k * 0.25));
    const float cc = (quarter & 1) ? s : c, ss = (quarter & 1) ? c : s;
    return {factor * ((quarter == 1 || quarter == 2) ? -cc : cc), factor * ((quarter & 2) ? -ss : ss)};
}

// N neighbouring pairs' turns; the angles that are far are looked for once.
template <int N>
__device__ __forceinline__ void turns_of(const double position, const double *freq, const float factor, Turn (&out)[N])
{
    bool far = false;
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = turn_by<false>(position, freq[j], factor, far);
    if (far) {
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = turn_by<true>(position, freq[j], factor, far);
    }
}

__device__ __forceinline__ double position_of(const void *positions, const int wide, const long long t)
{
    return wide ? (double)reinterpret_cast<const long long *>(positions)[t] : (double)reinterpret_cast<const int32_t *>(positions)[t];
}

// Eight consecutive elements as fp32.  They promise an element's alignment only.
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Raw {
    u32x4 w[DT == PTO_DT_FP32 ? 2 : 1];
    __device__ __forceinline__ void load(const void *base, const long long at)
    {
        if (DT == PTO_DT_FP32) {
            const float *p = static_cast<const float *>(base) + at;
            w[0] = *reinterpret_cast<const u32x4_a4 *>(p), w[DT == PTO_DT_FP32] = *reinterpret_cast<const u32x4_a4 *>(p + 4);
        } else {
            w[0] = *reinterpret_cast<const u32x4_a2 *>(static_cast<const uint16_t *>(base) + at);
        }
    }
};

template <int DT>
struct Eight {
    float v[8];
    __device__ __forceinline__ Eight() {}
    __device__ __forceinline__ explicit Eight(const Raw<DT> &r)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = r.w[0][i];
            if (DT == PTO_DT_FP32) {
                v[i] = __uint_as_float(a), v[4 + i] = __uint_as_float(r.w[DT == PTO_DT_FP32][i]);
            } else if (DT == PTO_DT_BF16) {
                v[2 * i] = __uint_as_float(a << 16), v[2 * i + 1] = __uint_as_float(a & 0xffff0000u);
            } else {
                const f16x2 h = __builtin_bit_cast(f16x2, a);
                v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
            }
        }
    }
    // (to be thrown out of the caches first: ordinary stores push out the rows that are still to be read, 28 us to 31)
    __device__ __forceinline__ void store(void *base, const long long at) const
    {
        if (DT == PTO_DT_FP32) {
            u32x4_a4 *p = reinterpret_cast<u32x4_a4 *>(static_cast<float *>(base) + at);
            u32x4_a4 a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[4 + i]);
            __builtin_nontemporal_store(a, p);
            __builtin_nontemporal_store(b, p + 1);
        } else {
            u32x4 a;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a[i] = DT == PTO_DT_BF16 ? pack_bf16x2(v[2 * i], v[2 * i + 1]) : pack_f16x2(v[2 * i], v[2 * i + 1]);
            __builtin_nontemporal_store((u32x4_a2)a, reinterpret_cast<u32x4_a2 *>(static_cast<uint16_t *>(base) + at));
        }
    }
};

template <int DT>
__device__ __forceinline__ void copy_one(const void *in, const long long from, void *out, const long long to)
{
    if (DT == PTO_DT_FP32)
        static_cast<uint32_t *>(out)[to] = static_cast<const uint32_t *>(in)[from];
    else
        static_cast<uint16_t *>(out)[to] = static_cast<const uint16_t *>(in)[from];
}

// A thread makes four neighbouring pairs' cosines and sines of one token.  A few microseconds of latency at any size met here.
template <int DT>
__global__ __launch_bounds__(256) void rotary_tables_kernel(const RotaryTablesParams p)
{
    const int quads = p.pairs / 4;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long t = i / quads;
    if (t >= p.T) return;
    const int pair = 4 * (int)(i - t * quads);
    const double n = position_of(p.positions, p.wide, t);
    float c[4], s[4];
    Turn turn[4];
    turns_of(n, p.freq + pair, p.factor, turn);
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = turn[j].c, s[j] = turn[j].s;
    const long long at = t * 2 * p.pairs + pair;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (DT == PTO_DT_FP32) {
            float *co = static_cast<float *>(p.cos) + at + h * p.pairs, *so = static_cast<float *>(p.sin) + at + h * p.pairs;
            u32x4_a4 x, y;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __float_as_uint(c[j]), y[j] = __float_as_uint(s[j]);
            *reinterpret_cast<u32x4_a4 *>(co) = x;
            *reinterpret_cast<u32x4_a4 *>(so) = y;
        } else {
            uint16_t *co = static_cast<uint16_t *>(p.cos) + at + h * p.pairs, *so = static_cast<uint16_t *>(p.sin) + at + h * p.pairs;
            constexpr bool B = DT == PTO_DT_BF16;
            *reinterpret_cast<u32x2_a2 *>(co) = u32x2{B ? pack_bf16x2(c[0], c[1]) : pack_f16x2(c[0], c[1]), B ? pack_bf16x2(c[2], c[3]) : pack_f16x2(c[2], c[3])};
            *reinterpret_cast<u32x2_a2 *>(so) = u32x2{B ? pack_bf16x2(s[0], s[1]) : pack_f16x2(s[0], s[1]), B ? pack_bf16x2(s[2], s[3]) : pack_f16x2(s[2], s[3])};
        }
    }
}

// A row (a token's head) is a group of LPR lanes of one wave, eight pairs to a lane, and a workgroup's 256 / LPR groups are heads of one token
// or, where a token has fewer, tokens side by side.  Their turns are made once, in LDS, while the rows are on their way; every lane's
// loads precede its group's stores, so a row may be turned where it lies whatever its layout.
// Bound by memory: 64 of 192 channels of 4096 tokens of 128 heads and a shared key, bf16, 135 MB in 27.1 us = 5.0 TB/s, what a plain copy
// reaches.  Whole heads that are turned out of place are not: their other channels are copied one element to a lane, 4096 tokens of 128 heads
// of 192 channels and a key, 406 MB, in 235 us, where a copy's rate gives 80 (in place, where nothing is copied, 30).  Four tokens of a head to a lane, one after the other, 28.7 us; results stored as if they were wanted soon 3 us more; the keys'
// workgroups in front of all of the queries' 31.4.  One head of a token after the other, 16384 tokens of 8 heads: 15.2 us, side by side 6.5.
template <int DT, int LPR>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p)
{
    constexpr int ROWS = 256 / LPR;
    __shared__ Turn turns[ROWS * 8 * LPR];
    const int tid = threadIdx.x;
    const int parts = p.side[0].parts + p.side[1].parts, at = (int)(blockIdx.x % (unsigned)parts);    // (a token's heads side by side)
    const bool key = at >= p.side[0].parts;
    const RotarySide &s = p.side[key ? 1 : 0];
    const int part = at - (key ? p.side[0].parts : 0);
    const long long t0 = (long long)(blockIdx.x / (unsigned)parts) * p.tokens;
    const int tokens = p.T - t0 < p.tokens ? (int)(p.T - t0) : p.tokens;

    const int lane = tid & (LPR - 1), group = tid / LPR;   // (a key of one head beside many heads leaves most groups idle)
    const int mine_t = p.tokens > 1 ? group / s.heads : 0, h = part * ROWS + group - mine_t * s.heads;
    const bool there = mine_t < tokens && h < s.heads;
    const bool mine = there && 8 * lane < p.pairs;         // (of a group some lanes may have no pairs)
    const int pair = 8 * lane;
    const bool half = p.layout == PTO_ROPE_HALF;
    const int first = half ? pair : 2 * pair, second = half ? pair + p.pairs : 2 * pair + 8;
    const bool halves = p.layout != PTO_ROPE_INTERLEAVED;  // of what is stored
    const int first_out = halves ? pair : 2 * pair, second_out = halves ? pair + p.pairs : 2 * pair + 8;
    const long long from = (t0 + mine_t) * s.in_t + h * s.in_h, to = (t0 + mine_t) * s.out_t + h * s.out_h;

    Raw<DT> ra, rb;
    if (mine) {
        ra.load(s.in, from + s.offset + first);
        rb.load(s.in, from + s.offset + second);
    }
    for (int i = tid; i < tokens * p.pairs; i += 256) {    // (the rows are on their way)
        const int t = i / p.pairs;
        Turn turn[1];
        turns_of(position_of(p.positions, p.wide, t0 + t), p.freq + (i - t * p.pairs), p.factor, turn);
        turns[i] = turn[0];
    }
    __syncthreads();
    if (!there) return;
    if (s.copies) {                                        // the channels around the part that turns
        const int rest = s.dim - 2 * p.pairs;
        for (int c = lane; c < rest; c += LPR) {
            const int ch = c < s.offset ? c : c + 2 * p.pairs;
            copy_one<DT>(s.in, from + ch, s.out, to + ch);
        }
    }
    if (!mine) return;
    Eight<DT> x(ra), y(rb), c, d;
    if (half) {
        c = x, d = y;
    } else {                                               // first and second members of the eight pairs
#pragma unroll
        for (int i = 0; i < 4; ++i) c.v[i] = x.v[2 * i], c.v[4 + i] = y.v[2 * i], d.v[i] = x.v[2 * i + 1], d.v[4 + i] = y.v[2 * i + 1];
    }
    const Turn *w = turns + mine_t * p.pairs + pair;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float u = c.v[i], v = d.v[i], co = w[i].c, si = w[i].s;
        c.v[i] = u * co - v * si;
        d.v[i] = v * co + u * si;
    }
    if (!halves) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[2 * i] = c.v[i], x.v[2 * i + 1] = d.v[i], y.v[2 * i] = c.v[4 + i], y.v[2 * i + 1] = d.v[4 + i];
        c = x, d = y;
    }
    c.store(s.out, to + s.offset + first_out);
    d.store(s.out, to + s.offset + second_out);
}

template <int DT, int LPR>
hipError_t rotary_with(RotaryParams p, hipStream_t stream)
{
    constexpr int rows = 256 / LPR;
    for (RotarySide &s : p.side) s.parts = (s.heads + rows - 1) / rows;
    // tokens side by side where a workgroup has room for them, as many as leave a workgroup to every compute unit
    const int most = p.side[0].heads > p.side[1].heads ? p.side[0].heads : p.side[1].heads;
    const long long room = rows / most, wide = p.T / p.cus, tokens = room < wide ? room : wide;
    p.tokens = tokens > 1 ? (int)tokens : 1;
    const long long grid = (p.T + p.tokens - 1) / p.tokens * (p.side[0].parts + p.side[1].parts);
    if (grid > 0x7fffffffll) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((rotary_kernel<DT, LPR>), dim3((unsigned)grid), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <int DT>
hipError_t rotary_of(const RotaryParams &p, hipStream_t stream)
{
    const int lanes = p.pairs / 8;
    return lanes <= 1 ? rotary_with<DT, 1>(p, stream) : lanes <= 2 ? rotary_with<DT, 2>(p, stream) : lanes <= 4 ? rotary_with<DT, 4>(p, stream)
         : lanes <= 8 ? rotary_with<DT, 8>(p, stream) : rotary_with<DT, 16>(p, stream);
}

}  // namespace

hipError_t rotary_tables_launch(const RotaryTablesParams &p, hipStream_t stream)
{
    const long long threads = p.T * (p.pairs / 4);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (p.dtype == PTO_DT_FP32) hipLaunchKernelGGL(rotary_tables_kernel<PTO_DT_FP32>, grid, dim3(256), 0, stream, p);
    else if (p.dtype == PTO_DT_BF16) hipLaunchKernelGGL(rotary_tables_kernel<PTO_DT_BF16>, grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(rotary_tables_kernel<PTO_DT_FP16>, grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t rotary_launch(const RotaryParams &p, hipStream_t stream)
{
    if (p.dtype == PTO_DT_FP32) return rotary_of<PTO_DT_FP32>(p, stream);
    if (p.dtype == PTO_DT_BF16) return rotary_of<PTO_DT_BF16>(p, stream);
    return rotary_of<PTO_DT_FP16>(p, stream);
}

}  // namespace pto
