// Block-format kernels: Q8_0 quantize / dequantize, GGUF Q8_0 and Q4_0 transcode,
// Q4_K and Q4_0 dequantize.  All are one-pass, HBM-bound maps over the tensor.
#include "device_common.h"

namespace rt {

static inline uint64_t align256(uint64_t n) { return (n + 255u) & ~(uint64_t)255u; }

// Quantizer::sint8_quantize (crates/ratchet-core/src/quant.rs:26-79).
// One lane per group of 32: d = max|x| / 127, q = round-half-away(x / d);
// a zero group gives d = 0 and x/d = NaN, which the reference's `as i32`
// turns into 0.
__global__ __launch_bounds__(256) void quantize_q8_0_kernel(const float *__restrict__ src, uint64_t ngroups,
                                                            uint8_t *__restrict__ qs, float *__restrict__ scales) {
    const uint64_t g = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (g >= ngroups) return;
    const float4_t *x4 = (const float4_t *)(src + g * 32);
    float x[32];
#pragma unroll
    for (int v = 0; v < 8; v++) {
        float4_t t = x4[v];
#pragma unroll
        for (int i = 0; i < 4; i++) x[4 * v + i] = t[i];
    }
    float amax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 32; i++) amax = fmaxf(amax, fabsf(x[i]));
    const float d = amax / 127.0f; // IEEE division, as the reference's f32 `/`
    uint32_t packed[8];
#pragma unroll
    for (int w = 0; w < 8; w++) {
        uint32_t pk = 0;
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const float r = roundf(x[4 * w + b] / d); // half away from zero
            int q = 0;
            if (!isnan(r)) q = (int)fminf(fmaxf(r, -2147483648.0f), 2147483520.0f);
            pk |= (uint32_t)(q & 0xFF) << (8 * b);
        }
        packed[w] = pk;
    }
    uint4_t *dst = (uint4_t *)(qs + g * 32);
    dst[0] = uint4_t{packed[0], packed[1], packed[2], packed[3]};
    dst[1] = uint4_t{packed[4], packed[5], packed[6], packed[7]};
    scales[g] = d;
}

__global__ void zero_bytes_kernel(uint8_t *p, uint64_t n) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) p[i] = 0;
}

// Quantizer::sint8_dequantize (quant.rs:81-124); ST = float (Q8_0F) or f16 (Q8_0H).
template <typename ST>
__global__ __launch_bounds__(256) void dequantize_q8_0_kernel(const uint8_t *__restrict__ qs,
                                                              const ST *__restrict__ scales, uint64_t nchunks,
                                                              float *__restrict__ dst) {
    const uint64_t c = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; // 16 weights per lane
    if (c >= nchunks) return;
    const uint4_t w = *(const uint4_t *)(qs + c * 16);
    const float d = to_f32(scales[c >> 1]);
    float4_t *o = (float4_t *)(dst + c * 16);
#pragma unroll
    for (int v = 0; v < 4; v++) {
        float4_t r;
#pragma unroll
        for (int b = 0; b < 4; b++) r[b] = (float)(int8_t)(w[v] >> (8 * b)) * d;
        o[v] = r;
    }
}

// ggml dequantize_row_q4_K; one lane per (super-block, 64-weight chunk).
__global__ __launch_bounds__(256) void dequantize_q4k_kernel(const uint8_t *__restrict__ blocks, uint64_t nchunks,
                                                             float *__restrict__ dst) {
    const uint64_t t = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= nchunks) return;
    const uint64_t sbi = t >> 2;
    const int c = (int)(t & 3);
    const uint8_t *blk = blocks + sbi * 144;
    const uint4_t hdr = *(const uint4_t *)blk;
    half2_t dm = __builtin_bit_cast(half2_t, hdr[0]);
    const float d = (float)dm[0], dmin = (float)dm[1];
    uint8_t sbytes[12];
#pragma unroll
    for (int i = 0; i < 12; i++) sbytes[i] = (uint8_t)(hdr[1 + (i >> 2)] >> (8 * (i & 3)));
    int sc0, mn0, sc1, mn1;
    q4k_scale_min(2 * c, sbytes, sc0, mn0);
    q4k_scale_min(2 * c + 1, sbytes, sc1, mn1);
    const float d0 = d * (float)sc0, m0 = dmin * (float)mn0;
    const float d1 = d * (float)sc1, m1 = dmin * (float)mn1;
    const uint4_t *q4 = (const uint4_t *)(blk + 16 + 32 * c);
    float *y = dst + sbi * 256 + 64 * c;
#pragma unroll
    for (int v = 0; v < 2; v++) {
        const uint4_t q = q4[v];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint32_t byte = (q[i >> 2] >> (8 * (i & 3))) & 0xFFu;
            // d*sc*q and dmin*mn are exact in f32; only the subtraction rounds
            y[16 * v + i] = __fsub_rn(__fmul_rn(d0, (float)(byte & 0xFu)), m0);
            y[32 + 16 * v + i] = __fsub_rn(__fmul_rn(d1, (float)(byte >> 4)), m1);
        }
    }
}

// GGUFInterop::transcode (crates/ratchet-loader/src/gguf/dtype.rs:40-110);
// one lane per 34-byte block.  Blocks are only 2-byte aligned, so they are
// read as 17 halfwords.
template <typename ST>
__global__ __launch_bounds__(256) void transcode_q8_0_kernel(const uint16_t *__restrict__ blocks, uint64_t nblocks,
                                                             uint8_t *__restrict__ qs, ST *__restrict__ scales) {
    const uint64_t b = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= nblocks) return;
    const uint16_t *src = blocks + b * 17;
    const uint16_t dbits = src[0];
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = (uint32_t)src[1 + 2 * i] | ((uint32_t)src[2 + 2 * i] << 16);
    uint4_t *dst = (uint4_t *)(qs + b * 32);
    dst[0] = uint4_t{w[0], w[1], w[2], w[3]};
    dst[1] = uint4_t{w[4], w[5], w[6], w[7]};
    if constexpr (sizeof(ST) == 2) {
        ((uint16_t *)scales)[b] = dbits;
    } else {
        scales[b] = (float)__builtin_bit_cast(half_t, dbits);
    }
}

// Q4_0 dequantize: one lane per dword, eight values.
__global__ __launch_bounds__(256) void dequantize_q40_kernel(const uint32_t *__restrict__ codes, const half_t *__restrict__ scales, uint64_t ndwords,
                                                             float *__restrict__ dst) {
    const uint64_t t = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= ndwords) return;
    const half8_t q = q40_codes(codes[t]);
    const float d = (float)scales[t >> 2];
    float4_t *o = (float4_t *)(dst + 8 * t);
#pragma unroll
    for (int v = 0; v < 2; v++) {
        float4_t r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = (float)q[4 * v + i] * d;
        o[v] = r;
    }
}

// GGUF Q4_0 (block_q4_0 of ggml, named but not loaded by the reference: crates/ratchet-loader/src/lib.rs:35-101): 18 bytes {f16 d; u8 qs[16]},
// qs[j] = value j in its low nibble, value j + 16 in its high one.  One lane per block: the nibbles of eight values into one dword, even
// values first (q40_codes).
__device__ __forceinline__ uint32_t q40_gather(uint32_t n) { // bytes 0x0v of values 0..3 -> nibbles 0, 4, 1, 5
    return (n & 0xFu) | ((n >> 12) & 0xF0u) | ((n << 8) & 0xF0000u) | ((n >> 4) & 0xF00000u);
}
__global__ __launch_bounds__(256) void transcode_q40_kernel(const uint16_t *__restrict__ blocks, uint64_t nblocks, uint8_t *__restrict__ codes,
                                                            uint16_t *__restrict__ scales) {
    const uint64_t b = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= nblocks) return;
    const uint16_t *src = blocks + b * 9;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)src[1 + 2 * i] | ((uint32_t)src[2 + 2 * i] << 16);
    uint4_t o;
#pragma unroll
    for (int u = 0; u < 4; u++) { // values 8 u .. + 7: bytes 8 (u % 2) .. + 7, low nibbles for u < 2
        const uint32_t a = (u < 2 ? w[2 * (u & 1)] : w[2 * (u & 1)] >> 4) & 0x0F0F0F0Fu;
        const uint32_t c = (u < 2 ? w[2 * (u & 1) + 1] : w[2 * (u & 1) + 1] >> 4) & 0x0F0F0F0Fu;
        o[u] = q40_gather(a) | (q40_gather(c) << 8);
    }
    *(uint4_t *)(codes + b * 16) = o;
    scales[b] = src[0];
}

static inline unsigned blocks_for(uint64_t n, unsigned threads) { return (unsigned)((n + threads - 1) / threads); }

static void zero_padding(uint8_t *base, uint64_t from, uint64_t to, hipStream_t stream) {
    if (to > from) hipLaunchKernelGGL(zero_bytes_kernel, dim3(1), dim3(256), 0, stream, base + from, to - from);
}

hipError_t launch_quantize_q8_0(const float *src, uint64_t numel, void *dst, hipStream_t stream) {
    if (numel == 0) return hipSuccess;
    const uint64_t ng = numel / 32, soff = align256(numel);
    uint8_t *d = (uint8_t *)dst;
    hipLaunchKernelGGL(quantize_q8_0_kernel, dim3(blocks_for(ng, 256)), dim3(256), 0, stream, src, ng, d,
                       (float *)(d + soff));
    zero_padding(d, numel, soff, stream);
    zero_padding(d, soff + ng * 4, soff + align256(ng * 4), stream);
    return hipGetLastError();
}

hipError_t launch_dequantize(int dtype, const void *src, uint64_t numel, float *dst, hipStream_t stream) {
    if (numel == 0) return hipSuccess;
    const uint8_t *s = (const uint8_t *)src;
    if (dtype == RT_Q8_0F || dtype == RT_Q8_0H) {
        const uint64_t nch = numel / 16, soff = align256(numel);
        if (dtype == RT_Q8_0F)
            hipLaunchKernelGGL((dequantize_q8_0_kernel<float>), dim3(blocks_for(nch, 256)), dim3(256), 0, stream, s,
                               (const float *)(s + soff), nch, dst);
        else
            hipLaunchKernelGGL((dequantize_q8_0_kernel<half_t>), dim3(blocks_for(nch, 256)), dim3(256), 0, stream, s,
                               (const half_t *)(s + soff), nch, dst);
    } else if (dtype == RT_Q4_K) {
        const uint64_t nch = numel / 64;
        hipLaunchKernelGGL(dequantize_q4k_kernel, dim3(blocks_for(nch, 256)), dim3(256), 0, stream, s, nch, dst);
    } else if (dtype == RT_Q4_0) {
        hipLaunchKernelGGL(dequantize_q40_kernel, dim3(blocks_for(numel / 8, 256)), dim3(256), 0, stream, (const uint32_t *)s,
                           (const half_t *)(s + q40_scale_offset(numel)), numel / 8, dst);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_transcode_gguf_q8_0(const void *blocks, uint64_t n_blocks, int dst_dtype, void *dst,
                                      hipStream_t stream) {
    if (n_blocks == 0) return hipSuccess;
    const uint64_t numel = n_blocks * 32, soff = align256(numel);
    uint8_t *d = (uint8_t *)dst;
    const uint64_t ssz = dst_dtype == RT_Q8_0H ? 2 : 4;
    if (dst_dtype == RT_Q8_0H)
        hipLaunchKernelGGL((transcode_q8_0_kernel<half_t>), dim3(blocks_for(n_blocks, 256)), dim3(256), 0, stream,
                           (const uint16_t *)blocks, n_blocks, d, (half_t *)(d + soff));
    else if (dst_dtype == RT_Q8_0F)
        hipLaunchKernelGGL((transcode_q8_0_kernel<float>), dim3(blocks_for(n_blocks, 256)), dim3(256), 0, stream,
                           (const uint16_t *)blocks, n_blocks, d, (float *)(d + soff));
    else
        return hipErrorInvalidValue;
    zero_padding(d, numel, soff, stream);
    zero_padding(d, soff + n_blocks * ssz, soff + align256(n_blocks * ssz), stream);
    return hipGetLastError();
}

hipError_t launch_transcode_gguf_q4_0(const void *blocks, uint64_t n_blocks, void *dst, hipStream_t stream) {
    if (n_blocks == 0) return hipSuccess;
    const uint64_t nb = n_blocks * 16, soff = q40_scale_offset(n_blocks * 32);
    uint8_t *d = (uint8_t *)dst;
    hipLaunchKernelGGL(transcode_q40_kernel, dim3(blocks_for(n_blocks, 256)), dim3(256), 0, stream, (const uint16_t *)blocks, n_blocks, d,
                       (uint16_t *)(d + soff));
    zero_padding(d, nb, soff, stream);
    zero_padding(d, soff + n_blocks * 2, soff + align256(n_blocks * 2), stream);
    return hipGetLastError();
}

} // namespace rt
