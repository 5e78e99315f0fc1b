// Q4_0 weights x up to 64 f16 activation rows (decode steps of one or many sequences): one pass over the weight on the matrix cores.
//
//   y[j, i] = act(sum_b d[i, b] * sum_{k in b} (q[i, k] - 8) x[j, k] + bias)        b: blocks of 32 of K
//
// v_mfma_f32_16x16x32_f16 contracts exactly one block for 16 weight rows and 16 activation rows.  The codes enter it unscaled (q - 8 is exact
// in f16), the block's sum is scaled by d in f32: no weight is rounded.  A lane's operand of it is one dword of codes (values
// 8 g .. + 7 of the block, g = lane / 16), which would make 16-byte pieces of 16 rows out of every load.  Instead lane group g loads the whole 16 bytes
// of block 4 c + g of its row, 64 contiguous bytes of a row per load instruction, and a 4 x 4 transposition among the lane groups (two
// v_permlane16_swap and two v_permlane32_swap for 512 weights' dwords) leaves dword g of block 4 c + t in register t.
//
// A result register holds one weight row (lane % 16) and activation row 4 (lane / 16) + r, so a lane needs one scale per block and one fused
// multiply-add per activation row that it holds.  Up to 4 (8) activation rows are put at MFMA rows 4 j (4 j, 4 j + 1), where one register (two)
// holds all of them.  More than 16 take further MFMAs on the same decoded weights.
//
// A workgroup owns 16 weight rows; its wavefronts share K in chunks of four blocks dealt out in turn, and add up their sums through LDS in a fixed order.
#include "device_common.h"

#include <algorithm>

namespace rt {

struct GemvQ40Args {
    const uint8_t *codes;
    const half_t *scales;
    const half_t *X;
    const half_t *bias;
    half_t *out;
    int64_t M, N, K; // weight rows, activation rows
    int64_t a_stack, b_stack;
    int64_t b_bs, b_js;
    int64_t o_bs, o_is, o_js;
    int has_bias, bias_on_rows, act;
    int waves; // wavefronts of a workgroup
};

typedef uint16_t ushort4_a2 __attribute__((ext_vector_type(4), aligned(2)));

// lane group g's register t <- lane group t's register g
__device__ __forceinline__ void q40_transpose(uint4_t &v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v[0], v[1], false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(v[2], v[3], false, false);
    const auto c = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
    v = uint4_t{c[0], d[0], c[1], d[1]};
}

// MT: groups of 16 activation rows; VPR: result registers in use (1, 2 or 4; 4 with MT > 1); U: chunks in flight
template <int MT, int VPR, int U> __global__ __launch_bounds__(1024) void gemv_q40_kernel(GemvQ40Args g) {
    extern __shared__ __attribute__((aligned(16))) float red[]; // [waves][MT][VPR][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, fg = lane >> 4;
    const int64_t s = blockIdx.y, i0 = (int64_t)blockIdx.x * 16;
    const int64_t row = (g.a_stack == 1 ? 0 : s) * g.M + min(i0 + r, g.M - 1); // (a row past the end repeats the last and is not stored)
    const int nb = (int)(g.K >> 5), full = nb >> 2; // blocks, chunks of four blocks
    const uint8_t *wp = g.codes + row * (g.K >> 1) + 16 * fg;
    const half_t *sp = g.scales + row * nb;
    const half_t *xp[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int64_t j = 16 * m + (r >> 2) * VPR + min(r & 3, VPR - 1);
        xp[m] = g.X + (g.b_stack == 1 ? 0 : s) * g.b_bs + min(j, g.N - 1) * g.b_js + 8 * fg;
    }
    float acc[MT][VPR];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int v = 0; v < VPR; v++) acc[m][v] = 0.f;

    struct Chunk {
        uint4_t w;
        ushort4_a2 d;
        uint4_t x[MT][4];
    };
    auto load = [&](int c, Chunk &k) __attribute__((always_inline)) {
        k.w = *(const uint4_t *)(wp + 64 * (int64_t)c);
        k.d = *(const ushort4_a2 *)(sp + 4 * (int64_t)c);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < 4; t++) k.x[m][t] = *(const uint4_t *)(xp[m] + 128 * (int64_t)c + 32 * t);
    };
    auto block = [&](uint32_t w, uint16_t d, const uint4_t *x, int stride) __attribute__((always_inline)) {
        const half8_t q = q40_codes(w);
        const float df = (float)__builtin_bit_cast(half_t, d);
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float4_t p = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, x[m * stride]), q, float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int v = 0; v < VPR; v++) acc[m][v] = fmaf(df, p[v], acc[m][v]);
        }
    };
    auto multiply = [&](Chunk &k) __attribute__((always_inline)) {
        q40_transpose(k.w);
#pragma unroll
        for (int t = 0; t < 4; t++) block(k.w[t], k.d[t], &k.x[0][t], 4);
    };
    const int waves = g.waves;
    int c = wave;
    for (; c + (U - 1) * waves < full; c += U * waves) {
        Chunk k[U];
#pragma unroll
        for (int u = 0; u < U; u++) load(c + u * waves, k[u]);
#pragma unroll
        for (int u = 0; u < U; u++) multiply(k[u]);
    }
    for (; c < full; c += waves) {
        Chunk k;
        load(c, k);
        multiply(k);
    }
    if (c == full && (nb & 3)) { // up to three blocks behind the last whole chunk, for the wavefront whose turn it is
        const int left = nb & 3;
        uint4_t w = *(const uint4_t *)(wp + 64 * (int64_t)c + 16 * (min(fg, left - 1) - fg));
        q40_transpose(w);
#pragma unroll
        for (int t = 0; t < 3; t++) {
            if (t < left) {
                uint4_t x[MT];
#pragma unroll
                for (int m = 0; m < MT; m++) x[m] = *(const uint4_t *)(xp[m] + 128 * (int64_t)c + 32 * t);
                block(w[t], __builtin_bit_cast(uint16_t, sp[4 * (int64_t)c + t]), x, 1);
            }
        }
    }

    constexpr int PER = MT * VPR * 64;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int v = 0; v < VPR; v++) red[wave * PER + (m * VPR + v) * 64 + lane] = acc[m][v];
    __syncthreads();
    rt_with_act(g.act, [&](auto has_act) {
        for (int e = threadIdx.x; e < PER; e += blockDim.x) {
            const int l = e & 63, mv = e >> 6, m = mv / VPR, v = mv - m * VPR;
            const int64_t i = i0 + (l & 15), j = 16 * m + (l >> 4) * VPR + v;
            if (i < g.M && j < g.N) {
                float y = 0.f;
                for (int w = 0; w < waves; w++) y += red[w * PER + e];
                if (g.has_bias) y += (float)g.bias[g.bias_on_rows ? i : j];
                g.out[s * g.o_bs + i * g.o_is + j * g.o_js] = (half_t)rt_act_k<decltype(has_act)::value>(y);
            }
        }
    });
}

template <int MT, int VPR, int U> static hipError_t launch_q40(const GemvQ40Args &g, dim3 grid, hipStream_t stream) {
    const size_t lds = (size_t)g.waves * MT * VPR * 64 * sizeof(float);
    if (lds > 48 * 1024)
        if (const hipError_t e = ensure_lds_limit<&gemv_q40_kernel<MT, VPR, U>>(); e != hipSuccess) return e;
    hipLaunchKernelGGL((gemv_q40_kernel<MT, VPR, U>), grid, dim3(64 * g.waves), lds, stream, g);
    return hipGetLastError();
}

hipError_t launch_gemv_q40(const Problem &p, const void *A, const void *B, const void *bias, void *out, hipStream_t stream, const DeviceInfo &dev) {
    if (p.a_dt != RT_Q4_0 || p.act_dt != RT_F16 || p.N < 1 || p.N > kGemvQ40MaxCols || (p.b_ks != 1 && p.K != 1) || p.K < 32 || p.K % 32 != 0) return hipErrorNotSupported;
    if (p.stacks > 65535 || p.K > 0x3fffffff || (p.M + 15) / 16 > 0x3fffff) return hipErrorNotSupported; // (a grid's threads along an axis are fewer than 2^32)
    if (((uintptr_t)A & 15u) || ((uintptr_t)B & 15u) || (p.b_js * 2) % 16 || (p.b_bs * 2) % 16) return hipErrorNotSupported;
    GemvQ40Args g{};
    g.codes = (const uint8_t *)A;
    g.scales = (const half_t *)((const uint8_t *)A + q40_scale_offset((uint64_t)p.a_stack * p.M * p.K));
    g.X = (const half_t *)B, g.bias = (const half_t *)bias, g.out = (half_t *)out;
    g.M = p.M, g.N = p.N, g.K = p.K;
    g.a_stack = p.a_stack, g.b_stack = p.b_stack, g.b_bs = p.b_bs, g.b_js = p.b_js;
    g.o_bs = p.o_bs, g.o_is = p.o_is, g.o_js = p.o_js;
    g.has_bias = p.has_bias, g.bias_on_rows = p.bias_on_rows, g.act = p.act;
    const int64_t tiles = (p.M + 15) / 16 * p.stacks, chunks = (p.K + 127) / 128;
    int waves = 4;
    while (waves < 16 && tiles * waves < 8 * (int64_t)dev.num_cus && chunks >= 4 * waves) waves *= 2;
    g.waves = (int)std::min<int64_t>(waves, chunks);
    const dim3 grid((unsigned)((p.M + 15) / 16), (unsigned)p.stacks);
    if (p.N <= 4) return launch_q40<1, 1, 4>(g, grid, stream);
    if (p.N <= 8) return launch_q40<1, 2, 4>(g, grid, stream);
    if (p.N <= 16) return launch_q40<1, 4, 4>(g, grid, stream);
    if (p.N <= 32) return launch_q40<2, 4, 2>(g, grid, stream);
    if (p.N <= 48) return launch_q40<3, 4, 1>(g, grid, stream);
    return launch_q40<4, 4, 1>(g, grid, stream);
}

} // namespace rt
