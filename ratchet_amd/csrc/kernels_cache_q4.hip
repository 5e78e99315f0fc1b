// A key/value cache held in 4-bit blocks: the write that quantizes new rows into it.
//
// Per block of 32 values of a row (the last may have 16): m the value of largest magnitude, the first of equals, t = |m| / 8,
//   d = -sign(m) * min(r(t), 8160),  r: rounded to eight significant bits, and to multiples of 2^-24,
//   q = clamp(floor(x / d + 8.5), 0, 15)   (d = 0: 8),   the value held: d * (q - 8).
// Eight significant bits of d and three of q - 8 (or a power of two) fit an f16, so the values held are f16 numbers and a reader may scale codes in f16
// without a rounding; m itself is met to 2^-8 from 2^-14 up (the limit included: 65504 is held as 65280) and to 2^-22 below.  A block with a NaN or an infinity gets d = NaN.
//
// The quotient is x * rcp(d) here.  Where x / d is not half way between two codes it is at least 2^-12 away from that: x has 11 significant bits
// and d eight, |x| >= |d| / 2 there, so 2 x - (2 n + 1) d is a multiple of 2^-3 units of d's last place, and 2 |d| is at most 510 of them.  (Where d is k < 256 times 2^-24, x is a
// multiple of 2^-24 too, and the distance at least 1 / (2 k).)  |x / d| is below 12: about 8, and up to 11 where d is 2^-24.  The product is within 2^-18 of it, the reciprocal
// being right to an ulp or so and the sum with 8.5 rounded to 2^-20, and 2^-15 added before the floor sends every half way up, as the formula does, and nothing else.
#include "device_common.h"

#include <algorithm>

namespace rt {

struct CacheQ4Args {
    uint8_t *codes[2];
    half_t *scales[2];
    const void *src[2];
    half_t *values[2];
    const int32_t *offsets; // per sequence, or NULL
    int64_t s_bs, s_hs, s_rs; // of the sources, in elements
    int heads, capacity, offset, len, D;
};

__device__ __forceinline__ uint32_t cq_quad_max(uint32_t v) { // over the four lanes of a block
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true)); // quad_perm 1 0 3 2
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true)); // quad_perm 2 3 0 1
}

// One thread per eight values of a row, four neighbouring threads per block; NB blocks a row.  blockIdx.y: sequence and head, z: keys or values.
template <typename T, int NB> __global__ __launch_bounds__(256) void cache_write_q4_kernel(CacheQ4Args g) {
    const uint32_t u = blockIdx.x * blockDim.x + threadIdx.x, i = u / (4 * NB), o = 8 * (u - i * (4 * NB)); // row, offset in it
    const int b = blockIdx.y / g.heads, h = blockIdx.y - b * g.heads, z = blockIdx.z;
    if (i >= (uint32_t)g.len) return; // (whole blocks: a quad stays together)
    const bool in = o < (uint32_t)g.D;
    uint4_t raw = {0, 0, 0, 0};
    if (in) {
        const T *src = (const T *)g.src[z] + b * g.s_bs + h * g.s_hs + i * g.s_rs + o;
        if constexpr (sizeof(T) == 2) {
            raw = *(const uint4_t *)src;
        } else {
            const float4_t lo = *(const float4_t *)src, hi = *(const float4_t *)(src + 4);
            raw = __builtin_bit_cast(uint4_t, half8_t{(half_t)lo[0], (half_t)lo[1], (half_t)lo[2], (half_t)lo[3], (half_t)hi[0], (half_t)hi[1], (half_t)hi[2],
                                                      (half_t)hi[3]});
        }
    }
    const half8_t x = __builtin_bit_cast(half8_t, raw);
    // |x| above, then how early it comes, then its sign: the largest such number is the block's m
    uint32_t key = 0;
    const uint32_t late = 31u - (o & 31u);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t v = (raw[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
        key = max(key, ((v & 0x7FFFu) << 6) | ((late - e) << 1) | (v >> 15));
    }
    key = cq_quad_max(key);
    const uint32_t mag = key >> 6;
    const float t = (float)__builtin_bit_cast(half_t, (uint16_t)mag) * 0.125f; // exact
    // to eight significant bits: as bfloat16, ties to even
    const uint32_t tb = __builtin_bit_cast(uint32_t, t);
    float d = __builtin_bit_cast(float, (tb + 0x7FFFu + ((tb >> 16) & 1u)) & 0xFFFF0000u);
    if (t < 0x1p-17f) d = (float)(half_t)t; // to multiples of 2^-24
    d = fminf(d, 8160.f);
    if (!(key & 1u)) d = -d;
    if (mag == 0) d = 0.f;
    if (mag >= 0x7C00u) d = __builtin_nanf("");
    const half_t dh = (half_t)d; // exact
    const float rd = __builtin_amdgcn_rcpf(d);
    uint32_t w = 0;
    half8_t val;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float q = floorf(fmaf((float)x[e], rd, 8.5f + 0x1p-15f));
        q = fminf(fmaxf(q, 0.f), 15.f);
        if (dh == (half_t)0.f || !(d == d)) q = 8.f;
        w |= (uint32_t)q << (4 * (e / 2 + 4 * (e & 1)));
        val[e] = (half_t)(q - 8.f) * dh;
    }
    if (!in) return;
    const int64_t bh = blockIdx.y;
    const int64_t r = (int64_t)g.offset + (g.offsets ? g.offsets[b] : 0) + i;
    if (r >= 0 && r < g.capacity) {
        constexpr int SR = NB == 3 ? 4 : NB; // scales a row takes
        const int64_t row = bh * g.capacity + r;
        *(uint32_t *)(g.codes[z] + row * (g.D >> 1) + (o >> 1)) = w;
        if ((o & 31u) == 0) g.scales[z][row * SR + (o >> 5)] = dh;
        if (SR > NB && o == 8) g.scales[z][row * SR + NB] = (half_t)0.f;
    }
    if (g.values[z]) *(half8_t *)(g.values[z] + (bh * g.len + i) * g.D + o) = val;
}

template <typename T> static hipError_t launch_cache_write_q4_t(const CacheQ4Args &g, int stacks, int tensors, hipStream_t st) {
    const int nb = (g.D + 31) / 32;
    const int64_t threads = (int64_t)g.len * nb * 4;
    const int block = (int)std::min<int64_t>(256, (threads + 63) / 64 * 64);
    const dim3 grid((unsigned)((threads + block - 1) / block), (unsigned)stacks, (unsigned)tensors);
    switch (nb) {
    case 1: hipLaunchKernelGGL((cache_write_q4_kernel<T, 1>), grid, dim3(block), 0, st, g); break;
    case 2: hipLaunchKernelGGL((cache_write_q4_kernel<T, 2>), grid, dim3(block), 0, st, g); break;
    case 3: hipLaunchKernelGGL((cache_write_q4_kernel<T, 3>), grid, dim3(block), 0, st, g); break;
    default: hipLaunchKernelGGL((cache_write_q4_kernel<T, 4>), grid, dim3(block), 0, st, g); break;
    }
    return hipGetLastError();
}

hipError_t launch_cache_write_q4(int src_dtype, void *k_cache, const void *k_src, void *v_cache, const void *v_src, const int64_t *strides, void *k_values,
                                 void *v_values, const int32_t *offsets, int batch, int heads, int capacity, int offset, int len, int head_dim,
                                 hipStream_t stream) {
    const uint64_t soff = cache_q4_scale_offset(batch, heads, capacity, head_dim);
    CacheQ4Args g{};
    g.codes[0] = (uint8_t *)k_cache, g.codes[1] = (uint8_t *)v_cache;
    g.scales[0] = (half_t *)((uint8_t *)k_cache + soff), g.scales[1] = (half_t *)((uint8_t *)v_cache + soff);
    g.src[0] = k_src, g.src[1] = v_src, g.values[0] = (half_t *)k_values, g.values[1] = (half_t *)v_values;
    g.offsets = offsets;
    g.s_bs = strides[0], g.s_hs = strides[1], g.s_rs = strides[2];
    g.heads = heads, g.capacity = capacity, g.offset = offset, g.len = len, g.D = head_dim;
    return src_dtype == RT_F16 ? launch_cache_write_q4_t<half_t>(g, batch * heads, v_cache ? 2 : 1, stream)
                               : launch_cache_write_q4_t<float>(g, batch * heads, v_cache ? 2 : 1, stream);
}

} // namespace rt
