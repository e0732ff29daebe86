// Writing rows of the quantised latent cache and reading them back, gfx950.
//
// A row is 512 int8 codes, one fp32 scale to 128 of them, and 64 bf16 rope channels.  Of a group v of 128 channels
//   steps = 127 * (1 / max |v|), code = rint(v * steps), scale = 1 / steps, value = bf16(code * scale),
// each an IEEE fp32 operation; the values are those that the attention multiplies.  (In this order torch evaluates 127 / max, so codes
// equal those of the rule written in torch.)  A caller whose rows are to be those that the MLA
// prolog writes asks for its steps, 127 / max in one rounding.  (20000 rows of normally distributed latents: 22 % of the scales differ
// between the two, by a bit or two, and of 10000 codes 3.9 in bf16, 0.9 in fp16, 0.01 in fp32, by one step; in bf16 one row in six holds
// such a code.  Codes of exact quotients are missed by 5.8 and 4.5 of 10000 in bf16.)  Both directions move bytes and nothing else bounds
// them.
#include <type_traits>

#include "common.h"
#include "prompt_device.h"
#include "prompt_ops.h"
#include "pypto_amd_sfa.h"

// quantisation is a fixed sequence of single roundings
#pragma clang fp contract(off)

namespace pto {
namespace {

typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// largest of an unsigned value over the sixteen lanes of a row, in each of them
__device__ __forceinline__ uint32_t row_max(uint32_t x)
{
    auto turned = [](const uint32_t v, auto ctrl) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xf, 0xf, true); };
    uint32_t y = turned(x, std::integral_constant<int, 0x128>{});       // row_ror:8
    x = x > y ? x : y;
    y = turned(x, std::integral_constant<int, 0x124>{});
    x = x > y ? x : y;
    y = turned(x, std::integral_constant<int, 0x122>{});
    x = x > y ? x : y;
    y = turned(x, std::integral_constant<int, 0x121>{});
    return x > y ? x : y;
}

template <int DT>
__device__ __forceinline__ float element(const void *base, const long long at)
{
    if (DT == PTO_DT_FP32) return static_cast<const float *>(base)[at];
    const uint16_t h = static_cast<const uint16_t *>(base)[at];
    return DT == PTO_DT_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
}

// A wave writes a token: eight latent channels to a lane, sixteen lanes to a scale.  All of a token's reads are on their way
// before the first is needed; the row's four stores follow a chain of two memory latencies.  8191 tokens, bf16, values back: 23 MB in 5.2 us
// (at a plain copy's rate 4.6); the values stored as if they were wanted soon 5.8.
template <int DT>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheWriteParams p)
{
    const int l = threadIdx.x & 63;
    const long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= p.T) return;
    const long long row = p.index[t];
    const float rope = element<DT>(p.rope, t * p.rope_t + l);
    float v[8];
    if (DT == PTO_DT_FP32) {
        const float *src = static_cast<const float *>(p.latent) + t * p.latent_t + 8 * l;
        const u32x4_a4 a = *reinterpret_cast<const u32x4_a4 *>(src), b = *reinterpret_cast<const u32x4_a4 *>(src + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
    } else {
        const u32x4 a = *reinterpret_cast<const u32x4_a2 *>(static_cast<const uint16_t *>(p.latent) + t * p.latent_t + 8 * l);
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
    // the bits of |v| order as the numbers do, infinities and then everything that is no number at the top
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
        most = most > a ? most : a;
    }
    most = row_max(most);
    const bool number = most < 0x7f800000u;
    const float steps = p.one_rounding ? __fdiv_rn(127.0f, __uint_as_float(most)) : 127.0f * (1.0f / __uint_as_float(most));
    // a group of zeros (or of values below 127 / FLT_MAX, whose steps would be infinite) is stored as zeros
    const bool zero = !(steps <= 3.4028235e38f);
    const float scale = number ? (zero ? 0.0f : 1.0f / steps) : __uint_as_float(0x7fc00000u);
    uint32_t code[2] = {0, 0}, value[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = zero || !number ? 0.0f : rintf(v[i] * steps);
        code[i >> 2] |= ((uint32_t)(int)x & 0xffu) << (8 * (i & 3));
        v[i] = x * scale;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) value[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    if (row >= 0 && row < p.cache.rows) {
        *reinterpret_cast<u32x2 *>(p.cache.nope + row * p.cache.nope_pitch + 8 * l) = u32x2{code[0], code[1]};
        *reinterpret_cast<uint16_t *>(p.cache.rope + row * p.cache.rope_pitch + 2 * l) = (uint16_t)pack_bf16x2(rope, rope);
        if ((l & 15) == 0) *reinterpret_cast<float *>(p.cache.scale + row * p.cache.scale_pitch + (l >> 2)) = scale;
    }
    if (p.values) __builtin_nontemporal_store((u32x4_a2)u32x4{value[0], value[1], value[2], value[3]}, reinterpret_cast<u32x4_a2 *>(p.values + t * p.values_t + 8 * l));
}

// A wave reads eight consecutive rows, two at a time: 32 lanes to a row, of either half of its latent eight channels to a lane (so that a store
// writes whole cache lines), four rope channels to sixteen of them.  The cache rows are looked up first, one to a lane: three latencies
// after one another, of the sequence's beginning, of its page and of the rows, all of whose loads are on their way before the first is stored.
// Bound by memory: 65536 rows 118 MB in 19.1 us = 6.2 TB/s (of which the caches hold a part); four batches of rows to a wave, so that a
// look-up serves 32, 20.3 us, and twice as slow for 1024 rows.
constexpr int READ_ROWS = 8;

__global__ __launch_bounds__(256) void cache_read_kernel(const CacheReadParams p)
{
    const int l = threadIdx.x & 63, half = l >> 5, i = l & 31;
    const long long r0 = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * READ_ROWS;
    if (r0 >= p.rows) return;
    const int s0 = sequence_of(p.cu, p.B, r0);
    if (s0 >= p.B) return;                                 // behind the last sequence
    int slot = -2;                                         // cache row of output row r0 + l; -1: no such row; -2: nothing to write
    if (l < READ_ROWS) {
        const long long r = r0 + l;
        int s = s0;
        while (s < p.B && p.cu[s + 1] <= r) ++s;
        if (r < p.rows && s < p.B && r >= p.cu[s]) {
            const long long at = r - p.cu[s] + (p.first ? p.first[s] : 0);
            slot = -1;
            if (at >= 0 && at < (long long)p.maxblk * p.bs) {
                const int block = (int)((uint64_t)at / (uint32_t)p.bs);
                const long long page = p.bt[(long long)s * p.maxblk + block];
                const long long row = page * p.bs + (at - (long long)block * p.bs);
                if (page >= 0 && row < p.cache.rows) slot = (int)row;
            }
        }
    }
    constexpr int N = READ_ROWS / 2;
    int from[N];
    u32x2 code[N][2], rope[N];
    f32x4 scales[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        from[j] = __shfl(slot, 2 * j + half);
        code[j][0] = code[j][1] = rope[j] = u32x2{0, 0};
        scales[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (from[j] >= 0) {
            const uint8_t *row = p.cache.nope + (long long)from[j] * p.cache.nope_pitch;
            code[j][0] = *reinterpret_cast<const u32x2 *>(row + 8 * i);
            code[j][1] = *reinterpret_cast<const u32x2 *>(row + 256 + 8 * i);
            scales[j] = *reinterpret_cast<const f32x4 *>(p.cache.scale + (long long)from[j] * p.cache.scale_pitch);
            if (i < 16) rope[j] = *reinterpret_cast<const u32x2 *>(p.cache.rope + (long long)from[j] * p.cache.rope_pitch + 8 * i);
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (from[j] < -1) continue;
        const long long r = r0 + 2 * j + half;
        uint16_t *dst = p.latent + r * p.latent_t + 8 * i;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float scale = i < 16 ? scales[j][2 * h] : scales[j][2 * h + 1];
            u32x4 out;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t w = code[j][h][k >> 1] >> (16 * (k & 1));
                out[k] = pack_bf16x2((float)(int8_t)(w & 0xff) * scale, (float)(int8_t)((w >> 8) & 0xff) * scale);
            }
            __builtin_nontemporal_store((u32x4_a2)out, reinterpret_cast<u32x4_a2 *>(dst + 256 * h));
        }
        if (i < 16) __builtin_nontemporal_store((u32x2_a2)rope[j], reinterpret_cast<u32x2_a2 *>(p.rope + r * p.rope_t + 4 * i));
    }
}

}  // namespace

hipError_t cache_write_launch(const CacheWriteParams &p, hipStream_t stream)
{
    const dim3 grid((unsigned)((p.T + 3) / 4));
    if (p.dtype == PTO_DT_FP32) hipLaunchKernelGGL(cache_write_kernel<PTO_DT_FP32>, grid, dim3(256), 0, stream, p);
    else if (p.dtype == PTO_DT_BF16) hipLaunchKernelGGL(cache_write_kernel<PTO_DT_BF16>, grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(cache_write_kernel<PTO_DT_FP16>, grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t cache_read_launch(const CacheReadParams &p, hipStream_t stream)
{
    constexpr int rows = 4 * READ_ROWS;
    hipLaunchKernelGGL(cache_read_kernel, dim3((unsigned)((p.rows + rows - 1) / rows)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pto
