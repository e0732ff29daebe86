// Rotary positions, gfx950.
//
// Channel pair i of a token at position n turns by the angle n * freq[i].  The angle needs 64 bits (position 131071 in fp32
// leaves an angle 2^-7 of its bits after the point); it is reduced to the nearest quarter turn there, and what is left, at most
// pi/4, goes through the sine's and cosine's series in fp32, whose first left-out terms are below 2e-9.
#include "common.h"
#include "prompt_ops.h"
#include "pypto_amd_sfa.h"

namespace pto {
namespace {

struct Turn {
    float c, s;
};

__device__ __forceinline__ Turn turn_of(const double position, const double freq, const float factor)
{
    const double angle = position * freq;
    const double k = rint(angle * 0.63661977236758134308);                  // 2 / pi
    // pi / 2 as the sum of two doubles
    const double left = fma(-k, 6.123233995736766036e-17, fma(-k, 1.5707963267948965580, angle));
    const float x = (float)left, z = x * x;
    const float s = x + x * z * (-1.6666667e-1f + z * (8.3333333e-3f + z * (-1.9841270e-4f + z * 2.7557319e-6f)));
    const float c = 1.0f + z * (-0.5f + z * (4.1666667e-2f + z * (-1.3888889e-3f + z * 2.4801587e-5f)));
    const int quarter = (int)(k - 4.0 * floor(k * 0.25));
    const float cc = (quarter & 1) ? s : c, ss = (quarter & 1) ? c : s;
    return {factor * ((quarter == 1 || quarter == 2) ? -cc : cc), factor * ((quarter & 2) ? -ss : ss)};
}

__device__ __forceinline__ double position_of(const void *positions, const int wide, const long long t)
{
    return wide ? (double)reinterpret_cast<const long long *>(positions)[t] : (double)reinterpret_cast<const int32_t *>(positions)[t];
}

// Eight consecutive elements as fp32.  They promise an element's alignment only.
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Eight {
    float v[8];
    __device__ __forceinline__ void load(const void *base, const long long at)
    {
        if (DT == PTO_DT_FP32) {
            const float *p = static_cast<const float *>(base) + at;
            const u32x4_a4 a = *reinterpret_cast<const u32x4_a4 *>(p), b = *reinterpret_cast<const u32x4_a4 *>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4_a2 *>(static_cast<const uint16_t *>(base) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (DT == PTO_DT_BF16) {
                    v[2 * i] = __uint_as_float(a[i] << 16), v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
                } else {
                    const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)a[i]);
                    v[2 * i] = (float)h[0], v[2 * i + 1] = (float)h[1];
                }
            }
        }
    }
    __device__ __forceinline__ void store(void *base, const long long at) const
    {
        if (DT == PTO_DT_FP32) {
            float *p = static_cast<float *>(base) + at;
            u32x4_a4 a, b;
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[4 + i]);
            *reinterpret_cast<u32x4_a4 *>(p) = a;
            *reinterpret_cast<u32x4_a4 *>(p + 4) = b;
        } else {
            u32x4 a;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a[i] = DT == PTO_DT_BF16 ? pack_bf16x2(v[2 * i], v[2 * i + 1]) : pack_f16x2(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<u32x4_a2 *>(static_cast<uint16_t *>(base) + at) = a;
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
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const Turn a = turn_of(n, p.freq[pair + j], p.factor);
        c[j] = a.c, s[j] = a.s;
    }
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

// A workgroup makes the turns of a few tokens once, in LDS, and takes them through all heads, queries' and keys' rows one after
// the other.  A row is a group of LPR lanes of one wave, eight pairs to a lane: every lane's loads precede the row's
// stores, so a row may be turned where it lies whatever its layout.
template <int DT, int LPR>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p)
{
    __shared__ Turn turns[8 * ROT_MAX_PAIRS];              // at most eight tokens to a workgroup
    const int tid = threadIdx.x;
    const long long t0 = (long long)blockIdx.x * p.tokens_per_wg;
    const int tokens = p.T - t0 < p.tokens_per_wg ? (int)(p.T - t0) : p.tokens_per_wg;
    for (int i = tid; i < tokens * p.pairs; i += 256) {
        const int t = i / p.pairs;
        turns[i] = turn_of(position_of(p.positions, p.wide, t0 + t), p.freq[i - t * p.pairs], p.factor);
    }
    __syncthreads();

    const int lane = tid & (LPR - 1);
    const bool mine = 8 * lane < p.pairs;                  // (of a group some lanes may have no pairs)
    const int pair = mine ? 8 * lane : 0;
    const int heads = p.side[0].heads + p.side[1].heads;
    // this workgroup's share of every token's heads
    const int share = (heads + p.head_parts - 1) / p.head_parts;
    const int h_begin = blockIdx.y * share;
    const int h_end = h_begin + share < heads ? h_begin + share : heads;
    const int width = h_end - h_begin;
    if (width <= 0) return;
    const int rows = tokens * width;
    for (int r = tid / LPR; r < rows; r += 256 / LPR) {
        const int t = r / width;
        int h = h_begin + r - t * width;
        const bool key = h >= p.side[0].heads;
        const RotarySide &s = p.side[key ? 1 : 0];
        h -= key ? p.side[0].heads : 0;
        const long long from = (t0 + t) * s.in_t + h * s.in_h, to = (t0 + t) * s.out_t + h * s.out_h;
        Eight<DT> a, b;
        if (mine) {
            const long long at = from + s.offset;
            a.load(s.in, at + (p.layout == PTO_ROPE_HALF ? pair : 2 * pair));
            b.load(s.in, at + (p.layout == PTO_ROPE_HALF ? pair + p.pairs : 2 * pair + 8));
            if (p.layout != PTO_ROPE_HALF) {               // first and second halves of the eight pairs
                Eight<DT> x, y;
#pragma unroll
                for (int i = 0; i < 4; ++i) x.v[i] = a.v[2 * i], x.v[4 + i] = b.v[2 * i], y.v[i] = a.v[2 * i + 1], y.v[4 + i] = b.v[2 * i + 1];
                a = x, b = y;
            }
            const Turn *w = turns + t * p.pairs + pair;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = a.v[i], y = b.v[i], c = w[i].c, z = w[i].s;
                a.v[i] = x * c - y * z;
                b.v[i] = y * c + x * z;
            }
            if (p.layout == PTO_ROPE_INTERLEAVED) {
                Eight<DT> x, y;
#pragma unroll
                for (int i = 0; i < 4; ++i) x.v[2 * i] = a.v[i], x.v[2 * i + 1] = b.v[i], y.v[2 * i] = a.v[4 + i], y.v[2 * i + 1] = b.v[4 + i];
                a = x, b = y;
            }
        }
        if (s.copies) {                                    // the channels around the part that turns
            const int rest = s.dim - 2 * p.pairs;
            for (int c = lane; c < rest; c += LPR) {
                const int ch = c < s.offset ? c : c + 2 * p.pairs;
                copy_one<DT>(s.in, from + ch, s.out, to + ch);
            }
        }
        if (mine) {
            const long long at = to + s.offset;
            const bool halves = p.layout != PTO_ROPE_INTERLEAVED;
            a.store(s.out, at + (halves ? pair : 2 * pair));
            b.store(s.out, at + (halves ? pair + p.pairs : 2 * pair + 8));
        }
    }
}

template <int DT>
hipError_t rotary_of(const RotaryParams &p, const dim3 grid, hipStream_t stream)
{
    const int lanes = p.pairs / 8;
    if (lanes <= 1) hipLaunchKernelGGL((rotary_kernel<DT, 1>), grid, dim3(256), 0, stream, p);
    else if (lanes <= 2) hipLaunchKernelGGL((rotary_kernel<DT, 2>), grid, dim3(256), 0, stream, p);
    else if (lanes <= 4) hipLaunchKernelGGL((rotary_kernel<DT, 4>), grid, dim3(256), 0, stream, p);
    else if (lanes <= 8) hipLaunchKernelGGL((rotary_kernel<DT, 8>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((rotary_kernel<DT, 16>), grid, dim3(256), 0, stream, p);
    return hipGetLastError();
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
    const dim3 grid((unsigned)((p.T + p.tokens_per_wg - 1) / p.tokens_per_wg), (unsigned)p.head_parts);
    if (p.dtype == PTO_DT_FP32) return rotary_of<PTO_DT_FP32>(p, grid, stream);
    if (p.dtype == PTO_DT_BF16) return rotary_of<PTO_DT_BF16>(p, grid, stream);
    return rotary_of<PTO_DT_FP16>(p, grid, stream);
}

}  // namespace pto
