// Q4_0 weights x one or two f16 vectors: rows streamed from HBM, dot products on the vector unit.
//
//   y[j, i] = act(sum_b d[i, b] * sum_{k in b} (q[i, k] - 8) x[j, k] + bias)        b: blocks of 32 of K
//
// For so few vectors the matrix cores need a transposition and panels that every wavefront waits for, and decode steps are bound by how soon the weights are asked
// for.  Here a wavefront has four rows, sixteen lanes each, and a lane the blocks seg, seg + 16, .. of its share of K (up to five: 2560 values): one 16-byte load
// of codes (256 contiguous bytes of a row per four rows and load) and one of a scale for each, all requested before anything else.  The vector comes
// through LDS, where its 64-byte blocks are read in four pieces whose order depends on the block, so that no bank is met twice.  Where there are more groups of
// rows than wavefronts, the next group's weights are on their way while one is multiplied.  Thirteen instructions for eight weights: nine of
// q40_codes, exact, and four dot products; a block's sum is scaled in f32.  The sixteen lanes are joined by DPP, the wavefronts that share K through LDS, in a
// fixed order.
//
// With a bias, from HBM in a captured graph, 10240 x 2560 6.7 us, 51865 x 2560 17.1 (4.4 TB/s, near a copy's 5.1), 2560 x 10240 7.9, 2560 x 2560 3.9: the small ones are a launch,
// one trip to memory and 1 us of instructions.  Two vectors, with four more dot products for eight weights: 7.8, 21.6, 9.4 and 4.4.
#include "device_common.h"

#include <algorithm>

namespace rt {

struct RowdotQ40Args {
    const uint8_t *codes;
    const half_t *scales;
    const half_t *X;
    const half_t *bias;
    half_t *out;
    int64_t M, K, a_stack, b_stack, b_bs, b_js, o_bs, o_is, o_js;
    int N, has_bias, bias_on_rows, act;
    int wk;               // wavefronts that share K (the others of the workgroup have other rows)
    int64_t groups, step; // of four rows; those of a pass
};

template <int CTRL> __device__ __forceinline__ float q40_dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// NB: blocks of a lane; NV: vectors
template <int NB, int NV> __global__ __launch_bounds__(512, NV == 1 ? 4 : 3) void gemv_q40_rowdot_kernel(RowdotQ40Args g) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), threads = blockDim.x;
    const int wk = g.wk, wr = __builtin_amdgcn_readfirstlane(wave / wk), kc = wave - wr * wk;
    const int seg = lane & 15, nb = (int)(g.K >> 5), b0 = kc * (16 * NB) + seg;
    const int64_t s = blockIdx.y;
    const uint8_t *const codes = g.codes + (g.a_stack == 1 ? 0 : s) * g.M * (g.K >> 1);
    const half_t *const scales = g.scales + (g.a_stack == 1 ? 0 : s) * g.M * nb;
    struct Rows {
        uint4_t w[NB];
        half_t d[NB], bias;
    };
    const half_t *const from = g.has_bias ? g.bias : g.X; // (read in any case, so that the loads in flight are the same number)
    auto load = [&](int64_t group, Rows &k) __attribute__((always_inline)) { // (rows and blocks past the end repeat the last)
        const int64_t row = min(4 * group + (lane >> 4), g.M - 1);
        const uint8_t *const w = codes + row * (g.K >> 1);
        const half_t *const d = scales + row * nb;
#pragma unroll
        for (int i = 0; i < NB; i++) k.w[i] = *(const uint4_t *)(w + 16 * (uint32_t)min(b0 + 16 * i, nb - 1));
#pragma unroll
        for (int i = 0; i < NB; i++) k.d[i] = d[min(b0 + 16 * i, nb - 1)];
        k.bias = from[!g.has_bias ? 0 : g.bias_on_rows ? row : min(seg, NV - 1)];
    };
    const int64_t first = (int64_t)blockIdx.x * (threads / (64 * wk));
    Rows ring[2];
    load(first + wr, ring[0]);
    __builtin_amdgcn_sched_barrier(0);

    // ---- the vectors in LDS: piece p of block b at 4 b + (p + b / 4) % 4
    uint4_t *const xs = (uint4_t *)smem;
    const int xn = 64 * NB * wk; // pieces of a vector, to whole shares of K (what is behind its end is read and not used)
    const half_t *const X = g.X + (g.b_stack == 1 ? 0 : s) * g.b_bs;
    for (int e = t; e < 4 * nb; e += threads) {
#pragma unroll
        for (int j = 0; j < NV; j++) xs[xn * j + (e & ~3) + ((e + (e >> 4)) & 3)] = *(const uint4_t *)(X + j * g.b_js + 8 * e);
    }
    __syncthreads();
    int xo[4];
#pragma unroll
    for (int p = 0; p < 4; p++) xo[p] = 4 * b0 + ((p + (b0 >> 2)) & 3);
    float *const part = (float *)(xs + xn * NV); // [2][row group of the workgroup][share of K][4 rows][NV], where K is shared
    const uint32_t bias = q40_bias();

    auto multiply = [&](int64_t at, Rows &k, int buf) __attribute__((always_inline)) {
        asm volatile("" ::: "memory"); // (the vectors are read again for each group of rows: in registers they would leave room for half as many wavefronts)
        float acc[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) acc[j] = 0.f;
        // With two vectors a block's pieces are read while the block before it is multiplied, and no more: left alone the compiler reads them all first, in more registers
        // than there are.  With one that is what is wanted.
        half8_t x[2][NV][4];
        auto read = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NV; j++)
#pragma unroll
                for (int p = 0; p < 4; p++) x[i & 1][j][p] = __builtin_bit_cast(half8_t, xs[xn * j + xo[p] + 64 * i]);
        };
        if (NV > 1) read(0);
#pragma unroll
        for (int i = 0; i < NB; i++) {
            if (NV == 1) read(i);
            if (NV > 1 && i + 1 < NB) read(i + 1);
            if (NV > 1) __builtin_amdgcn_sched_barrier(0);
            float sum[NV][2];
#pragma unroll
            for (int j = 0; j < NV; j++) sum[j][0] = sum[j][1] = 0.f;
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const half8_t q = q40_codes(k.w[i][p], bias);
#pragma unroll
                for (int j = 0; j < NV; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        sum[j][c & 1] = __builtin_amdgcn_fdot2(half2_t{q[2 * c], q[2 * c + 1]}, half2_t{x[i & 1][j][p][2 * c], x[i & 1][j][p][2 * c + 1]}, sum[j][c & 1], false);
            }
            const bool in = b0 + 16 * i < nb;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                acc[j] = in ? fmaf((float)k.d[i], sum[j][0] + sum[j][1], acc[j]) : acc[j];
                if (NV > 1) asm volatile("" : "+v"(acc[j]));
            }
            if (NV > 1) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            acc[j] += q40_dpp<0x128>(acc[j]), acc[j] += q40_dpp<0x124>(acc[j]);
            acc[j] += q40_dpp<0x122>(acc[j]);
            acc[j] += q40_dpp<0x121>(acc[j]);
        }
        float y = acc[0]; // lane j of a row's sixteen has vector j
        if constexpr (NV == 2) y = seg == 1 ? acc[1] : acc[0];
        if (wk > 1) {
            float *const p = part + (buf * (threads >> 6) + wr * wk) * (4 * NV);
            if (seg < NV) p[kc * 4 * NV + (lane >> 4) * NV + seg] = y;
            __syncthreads();
            y = 0.f;
            if (seg < NV)
                for (int c = 0; c < wk; c++) y += p[c * 4 * NV + (lane >> 4) * NV + seg];
        }
        const int64_t row = 4 * at + (lane >> 4);
        if (kc == 0 && seg < NV && row < g.M) {
            if (g.has_bias) y += (float)k.bias;
            rt_with_act(g.act, [&](auto has_act) { y = rt_act_k<decltype(has_act)::value>(y); });
            g.out[s * g.o_bs + row * g.o_is + seg * g.o_js] = (half_t)y;
        }
    };
    // all wavefronts of a workgroup make the same passes
    int64_t at = first;
#pragma unroll 1
    for (; at + g.step < g.groups; at += 2 * g.step) {
        load(at + g.step + wr, ring[1]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(at + wr, ring[0], 0);
        __builtin_amdgcn_sched_barrier(0);
        load(at + 2 * g.step + wr, ring[0]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(at + g.step + wr, ring[1], 1);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (at < g.groups) multiply(at + wr, ring[0], 0);
}

template <int NB> static hipError_t launch_rowdot(const RowdotQ40Args &g, int wr, int64_t stacks, hipStream_t st) {
    const int waves = wr * g.wk, nv = g.N;
    const size_t lds = (size_t)1024 * NB * g.wk * nv + (g.wk > 1 ? (size_t)2 * waves * 4 * nv * sizeof(float) : 0);
    const dim3 grid((unsigned)(g.step / wr), (unsigned)stacks), block(64 * waves);
    if (nv == 1) {
        if (const hipError_t e = ensure_lds_limit<&gemv_q40_rowdot_kernel<NB, 1>>(); e != hipSuccess) return e;
        hipLaunchKernelGGL((gemv_q40_rowdot_kernel<NB, 1>), grid, block, lds, st, g);
    } else {
        if (const hipError_t e = ensure_lds_limit<&gemv_q40_rowdot_kernel<NB, 2>>(); e != hipSuccess) return e;
        hipLaunchKernelGGL((gemv_q40_rowdot_kernel<NB, 2>), grid, block, lds, st, g);
    }
    return hipGetLastError();
}

// One or two vectors and K up to 10240, which four wavefronts of five blocks a lane hold, four wavefronts a workgroup (all sharing K where that is long), two workgroups per compute unit (us without a bias for 10240 x 2560 / 51865 x 2560, one vector:
// two 6.6 / 16.6, three 7.0 / 17.4; eight wavefronts 7.1 / 17.9).  The matrix-core kernel at one and two vectors and this: 10240 x 2560 8.4 / 8.3 and 6.6 / 7.5, 2560 x 10240 9.4 / 9.4 and 7.5 /
// 10.0, 2560 x 2560 5.9 / 5.9 and 4.0 / 4.9, 51865 x 2560 21.5 / 21.8 and 16.6 / 20.4, 8192 x 8192 13.0 / 14.4 and 11.2 / 12.9, 640 x 1024 4.1 and 2.5; 4096 x 14336 12.4 / 12.4, here with six
// wavefronts that share K 12.2 / 20: nothing to be had past 10240.
hipError_t launch_gemv_q40_rowdot(const Problem &p, const void *A, const void *B, const void *bias, void *out, hipStream_t stream, const DeviceInfo &dev) {
    if (p.a_dt != RT_Q4_0 || p.act_dt != RT_F16 || p.N < 1 || p.N > 2 || p.b_ks != 1 || p.K < 32 || p.K % 32 != 0 || p.K > 10240) return hipErrorNotSupported;
    const int units = (int)((p.K / 32 + 15) / 16), wk = (units + 4) / 5, nb = (units + wk - 1) / wk;
    if (p.stacks > 65535 || (p.N > 1 && wk > 2 && p.M < 4096)) return hipErrorNotSupported;
    if (((uintptr_t)A & 15u) || ((uintptr_t)B & 15u) || (p.N > 1 && (p.b_js * 2) % 16) || (p.stacks > 1 && (p.b_bs * 2) % 16)) return hipErrorNotSupported;
    RowdotQ40Args g{};
    g.codes = (const uint8_t *)A;
    g.scales = (const half_t *)((const uint8_t *)A + q40_scale_offset((uint64_t)p.a_stack * p.M * p.K));
    g.X = (const half_t *)B, g.bias = (const half_t *)bias, g.out = (half_t *)out;
    g.M = p.M, g.K = p.K, g.N = (int)p.N;
    g.a_stack = p.a_stack, g.b_stack = p.b_stack, g.b_bs = p.b_bs, g.b_js = p.b_js;
    g.o_bs = p.o_bs, g.o_is = p.o_is, g.o_js = p.o_js;
    g.has_bias = p.has_bias, g.bias_on_rows = p.bias_on_rows, g.act = p.act;
    g.wk = wk, g.groups = (p.M + 3) / 4;
    const int wr = 4 / wk;
    const int64_t wgs = std::min<int64_t>((g.groups + wr - 1) / wr, (int64_t)2 * dev.num_cus);
    g.step = wgs * wr;
    switch (nb) {
    case 1: return launch_rowdot<1>(g, wr, p.stacks, stream);
    case 2: return launch_rowdot<2>(g, wr, p.stacks, stream);
    case 3: return launch_rowdot<3>(g, wr, p.stacks, stream);
    case 4: return launch_rowdot<4>(g, wr, p.stacks, stream);
    default: return launch_rowdot<5>(g, wr, p.stacks, stream);
    }
}

} // namespace rt
