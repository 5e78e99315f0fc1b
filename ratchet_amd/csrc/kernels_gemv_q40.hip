// Q4_0 weights x f16 activations on the matrix cores, one pass over the weight for 3 to 64 activation rows (decode steps of some sequences; one or two rows are
// kernels_gemv_q40_rowdot.hip's up to a K of 10240)
// and tiles of 32 for more (prompts that launch_gemm_nt leaves).
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
// A workgroup is wr x wk wavefronts: wr own 16 weight rows each, wk share K.  K goes in panels of wk units of 128 UC values: with UC = 4 a unit is 256 bytes of a row,
// four loads one behind the other (64 bytes at a time, a unit's worth of other rows between them, the same lines were fetched twice), and 32 bytes of its
// scales, one load, spread to the lane groups by swaps.  The panel's activations sit in LDS for all wr (two panels: the next one's are
// loaded while this one is multiplied); codes and scales are requested DEPTH panels ahead.  Nothing in the loop is conditional, so that the wait for the
// activations counts the weights' loads behind them and leaves them in flight.  The wk partial sums are added through LDS in a fixed order.
// A K-vector (16 bytes) v of activation row j of a panel is at slot v * NV + j of LDS, j exchanged within its 16 by 4 (v % 4): reads
// (16 rows of one vector by a lane group) and writes (four vectors of a row by neighbouring lanes) then meet no bank twice.
//
// Measured (weights from HBM, a captured graph, us): 10240 x 2560 at 4 / 16 / 32 / 64 rows 8.4 / 9.7 / 12.1 / 16.4, 2560 x 10240 9.4 / 15.0 / 26.8 / 27.1, 51865 x 2560
// 22 / 26 / 34 / 56 (16 rows: 3.0 TB/s).  The large ones are bound by the issue of the unpacking: with one row and no bias 20.5 us, without its loads 14, with nothing but its loads 19,
// and a kernel that only reads the codes 12 (5.5 TB/s).  The small ones by latency: a launch, one trip to HBM and the sum over K are 5.4 us at 2560 x 2560.
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
    int wr, wk;         // wavefronts along the weight rows, and that share K
    int vec_out;        // outputs along the weight rows are contiguous and start on 16 bytes
    int tiles_j, remap; // tiles of activation rows; whether workgroups are dealt to the XCDs in ranges
    int bias_at;        // bytes of LDS before the tile's biases
};

typedef uint64_t uint64_a2 __attribute__((aligned(2)));

// floats between activation rows of sums in LDS: a multiple of 4 that keeps a wavefront's four rows of 16 apart
__host__ __device__ constexpr int q40_ld(int rows) { return rows + 4; }

// MT: groups of 16 activation rows; VPR: result registers in use (1, 2 or 4; 4 with MT > 1); XI: pieces of a panel's activations per
// thread, at least NV UC / (4 wr); UC: chunks of 128 in a unit of K (4, or 2 where registers are short); DEPTH: panels of weights in flight
template <int MT, int VPR, int XI, int UC, int DEPTH> __global__ __launch_bounds__(MT > 1 || XI > 4 ? 512 : 1024) void gemv_q40_kernel(GemvQ40Args g) {
    constexpr int NV = MT == 1 ? 4 * VPR : 16 * MT; // activation rows of a tile: a power of two
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int WR = g.wr, wk = g.wk, wki = __builtin_amdgcn_readfirstlane(wave / WR), wr = wave - wki * WR;
    const int r = lane & 15, fg = lane >> 4;
    uint32_t id = blockIdx.x;
    if (g.remap) id = (id & 7) * (gridDim.x >> 3) + (id >> 3);
    const uint32_t ti = __builtin_amdgcn_readfirstlane(id / (uint32_t)g.tiles_j), tj = id - ti * (uint32_t)g.tiles_j;
    const int64_t s = blockIdx.y, i0 = ((int64_t)ti * WR + wr) * 16, j0 = (int64_t)tj * NV;
    const int nb = (int)(g.K >> 5); // blocks
    const int panels = ((nb + 4 * UC - 1) / (4 * UC) + wk - 1) / wk;

    // ---- this wavefront's weights: offsets in 32 bits from the first row of the tile
    const int64_t row0 = (g.a_stack == 1 ? 0 : s) * g.M + min(i0, g.M - 1);
    const uint8_t *const wp = g.codes + row0 * (g.K >> 1);
    const half_t *const sp = g.scales + row0 * nb;
    const uint32_t row = (uint32_t)(min(i0 + r, g.M - 1) - min(i0, g.M - 1)); // (a row past the end repeats the last and is not stored)
    const uint32_t wo = row * (uint32_t)(g.K >> 1), so = row * (uint32_t)nb;
    struct Unit {
        uint4_t w[UC];
        uint64_t d;
    };
    // this wavefront's unit of panel p (any: blocks past the end are the last one's codes with scales of 0)
    auto load = [&](int p, Unit &k) __attribute__((always_inline)) {
        const int b0 = 4 * UC * (p * wk + wki);
#pragma unroll
        for (int c = 0; c < UC; c++) k.w[c] = *(const uint4_t *)(wp + (wo + 16u * (uint32_t)min(b0 + 4 * c + fg, nb - 1)));
        k.d = *(const uint64_a2 *)(sp + (so + (uint32_t)min(b0 + 4 * (fg & (UC - 1)), nb - 4)));
    };
    // ---- the panels' activations: neighbouring threads have four K-vectors of a row, then the next row's
    const int threads = 64 * WR * wk, pieces = 16 * UC * NV * wk; // of a panel
    const half_t *const X = g.X + (g.b_stack == 1 ? 0 : s) * g.b_bs + j0 * g.b_js; // offsets in 32 bits from the first row of the tile
    const int jn = (int)min<int64_t>(g.N - j0, NV) - 1, js = (int)g.b_js, kv = (int)(g.K >> 3); // K-vectors of a row
    uint4_t *const Xs = (uint4_t *)smem;
    auto swizzle = [](int j, int v) { return NV >= 16 ? j ^ (4 * (v & 3)) : j; };
    uint4_t xr[XI];
    auto load_x = [&](int p) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < XI; i++) {
            const int e = i * threads + t, j = (e >> 2) & (NV - 1), v = p * 16 * UC * wk + (e >> 2) / NV * 4 + (e & 3);
            const uint4_t x = *(const uint4_t *)(X + ((uint32_t)(min(j, jn) * js) + 8 * (uint32_t)min(v, kv - 1)));
            xr[i] = j <= jn && v < kv ? x : uint4_t{0, 0, 0, 0};
        }
    };
    auto store_x = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < XI; i++) {
            const int e = i * threads + t, j = (e >> 2) & (NV - 1), v = (e >> 2) / NV * 4 + (e & 3);
            if (e < pieces) Xs[buf * pieces + v * NV + swizzle(j, v)] = xr[i];
        }
    };

    float acc[MT][VPR];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int v = 0; v < VPR; v++) acc[m][v] = 0.f;

    const int xrow = MT == 1 ? (r >> 2) * VPR + min(r & 3, VPR - 1) : r; // activation row of this lane's operand (of its 16)
    const int xoff = fg * NV + swizzle(xrow, fg);
    // A block's sums are folded into the accumulators behind the next block's MFMAs.  (The barriers keep it at that: left alone the compiler
    // decodes and multiplies every block of a panel at once, in more registers than there are.)
    float4_t part[MT];
    float scale = 0.f;
#pragma unroll
    for (int m = 0; m < MT; m++) part[m] = float4_t{0.f, 0.f, 0.f, 0.f};
    auto fold = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            asm volatile("" : "+v"(part[m])); // (all four registers until here: one reused sooner waits for the matrix cores)
#pragma unroll
            for (int v = 0; v < VPR; v++) {
                acc[m][v] = fmaf(scale, part[m][v], acc[m][v]);
                asm volatile("" : "+v"(acc[m][v])); // here, not gathered at the end of the panel with every block's sums kept until then
            }
        }
    };
    const uint32_t bias = q40_bias();
    auto multiply = [&](Unit &k, int p) __attribute__((always_inline)) {
        const int b0 = 4 * UC * (p * wk + wki);
        const int at = b0 + 4 * (fg & (UC - 1)); // lane group fg has the scales of chunk fg % UC: of blocks past the end 0
        const uint64_t ds = at < nb ? k.d >> (16 * (at - min(at, nb - 4))) : 0;
        uint32_t lo[UC], hi[UC]; // of blocks 0 1 and 2 3 of each chunk
        q40_spread<UC>((uint32_t)ds, lo), q40_spread<UC>((uint32_t)(ds >> 32), hi);
        const uint4_t *const x = Xs + (p & 1) * pieces + wki * 16 * UC * NV + xoff;
        half8_t xf[2][MT]; // a block's activations are read while the block before it is multiplied
#pragma unroll
        for (int m = 0; m < MT; m++) xf[0][m] = __builtin_bit_cast(half8_t, x[16 * m]);
#pragma unroll
        for (int c = 0; c < UC; c++) {
            if (b0 + 4 * c >= nb) break; // (uniform)
            q40_transpose(k.w[c]);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int n = 4 * c + b;
                if (n < 4 * UC - 1) {
#pragma unroll
                    for (int m = 0; m < MT; m++) xf[(n + 1) & 1][m] = __builtin_bit_cast(half8_t, x[(n + 1) * 4 * NV + 16 * m]);
                }
                const half8_t q = q40_codes(k.w[c][b], bias);
                float4_t now[MT];
#pragma unroll
                for (int m = 0; m < MT; m++) now[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[n & 1][m], q, float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                fold();
                scale = (float)__builtin_bit_cast(half2_t, b < 2 ? lo[c] : hi[c])[b & 1];
#pragma unroll
                for (int m = 0; m < MT; m++) part[m] = now[m];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    // the tile's biases, asked for with the first activations: behind the last sum they would be another trip to memory (2560 x 2560 at 4 rows 5.9 us, so 5.5; 10240 x 2560 8.4 and 7.9)
    half_t *const biases = (half_t *)(smem + g.bias_at);
    const half_t *const from = g.has_bias ? g.bias : g.X;
    const half_t bias_t = from[!g.has_bias ? 0 : g.bias_on_rows ? min((int64_t)ti * 16 * WR + t, g.M - 1) : min(j0 + t, g.N - 1)];
    // panel p: multiplied from ring[p % (DEPTH + 1)], while panel p + DEPTH's weights and panel p + 1's activations are requested
    Unit ring[DEPTH + 1];
    load_x(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < DEPTH; u++) load(u, ring[u]);
    __builtin_amdgcn_sched_barrier(0);
    store_x(0);
    if (t < max(16 * WR, NV)) biases[t] = bias_t;
    __syncthreads();
    auto panel = [&](int p, Unit &now, Unit &next) __attribute__((always_inline)) {
        load_x(p + 1);
        __builtin_amdgcn_sched_barrier(0);
        load(p + DEPTH, next);
        __builtin_amdgcn_sched_barrier(0);
        multiply(now, p);
        store_x((p + 1) & 1);
        __syncthreads();
    };
    int p = 0;
#pragma unroll 1
    for (; p + DEPTH < panels; p += DEPTH + 1) {
#pragma unroll
        for (int u = 0; u <= DEPTH; u++) panel(p + u, ring[u], ring[(u + DEPTH) % (DEPTH + 1)]);
    }
#pragma unroll
    for (int u = 0; u < DEPTH; u++)
        if (p + u < panels) {
            if (p + u + 1 < panels) load_x(p + u + 1);
            multiply(ring[u], p + u);
            if (p + u + 1 < panels) store_x((p + u + 1) & 1);
            __syncthreads();
        }
    fold();

    // ---- sums [share of K][activation row][weight row] through LDS; then the shares added, bias, activation, the one rounding, eight weight rows a thread
    const int ROWS = 16 * WR, LD = q40_ld(ROWS);
    float *const red = (float *)smem;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int v = 0; v < VPR; v++) red[(wki * NV + 16 * m + fg * VPR + v) * LD + wr * 16 + r] = acc[m][v];
    __syncthreads();
    const int64_t first = (int64_t)ti * ROWS;
    half_t *const out = g.out + s * g.o_bs;
    rt_with_act(g.act, [&](auto has_act) {
#pragma unroll 1
        for (int e = t; e < NV * (ROWS / 8); e += threads) {
            const int j = e / (ROWS / 8), i = 8 * (e - j * (ROWS / 8));
            if (j0 + j >= g.N || first + i >= g.M) continue;
            float y[8];
#pragma unroll
            for (int x = 0; x < 8; x++) y[x] = 0.f;
#pragma unroll 1
            for (int k = 0; k < wk; k++) {
                const float4_t *p = (const float4_t *)(red + (k * NV + j) * LD + i);
                const float4_t lo = p[0], hi = p[1];
#pragma unroll
                for (int x = 0; x < 4; x++) y[x] += lo[x], y[4 + x] += hi[x];
            }
            half8_t h;
            const int64_t left = g.M - first - i;
#pragma unroll
            for (int x = 0; x < 8; x++) {
                if (g.has_bias) y[x] += (float)biases[g.bias_on_rows ? i + x : j];
                h[x] = (half_t)rt_act_k<decltype(has_act)::value>(y[x]);
            }
            half_t *const o = out + (first + i) * g.o_is + (j0 + j) * g.o_js;
            if (g.vec_out && left >= 8) {
                *(half8_t *)o = h;
            } else {
#pragma unroll
                for (int x = 0; x < 8; x++)
                    if (x < left) o[x * g.o_is] = h[x];
            }
        }
    });
}

template <int MT, int VPR, int XI, int UC, int DEPTH> static hipError_t launch_q40(GemvQ40Args g, int64_t stacks, int wr, int wk, hipStream_t stream) {
    constexpr int NV = MT == 1 ? 4 * VPR : 16 * MT;
    if (4 * XI * wr < NV * UC) return hipErrorInvalidValue;
    g.wr = wr, g.wk = wk;
    const int64_t ti = (g.M + 16 * wr - 1) / (16 * wr), tj = (g.N + NV - 1) / NV;
    if (ti * tj > 0x3fffff) return hipErrorNotSupported; // (a grid's threads along an axis are fewer than 2^32)
    g.tiles_j = (int)tj, g.remap = tj > 1 && ti * tj % 8 == 0;
    const size_t panel = (size_t)NV * wk * UC * 256, x = g.K > 128 * UC * wk ? 2 * panel : panel, red = (size_t)wk * NV * q40_ld(16 * wr) * sizeof(float);
    g.bias_at = (int)std::max(x, red); // (whole 16 bytes)
    const size_t lds = (size_t)g.bias_at + std::max(16 * wr, NV) * sizeof(half_t);
    if (lds > 160 * 1024) return hipErrorNotSupported;
    if (lds > 48 * 1024)
        if (const hipError_t e = ensure_lds_limit<&gemv_q40_kernel<MT, VPR, XI, UC, DEPTH>>(); e != hipSuccess) return e;
    hipLaunchKernelGGL((gemv_q40_kernel<MT, VPR, XI, UC, DEPTH>), dim3((unsigned)(ti * tj), (unsigned)stacks), dim3(64 * wr * wk), lds, stream, g);
    return hipGetLastError();
}

// Wavefronts along the rows and along K, by the number of tiles of 16 weight rows (and 32 activation rows) and the units of 512 of K.  All (wr, wk) of up to
// 16 wavefronts were timed over M 320 .. 51865, K 512 .. 10240 and N 3, 8, 16, 32, 64, 160; the rules stay within 1 .. 12 % of the best there.  (Of (wr, wk): 33 to 64 rows take
// two tiles of 32, and every weight is unpacked for each; a tile of 64 was not built.)
// Few tiles: one row of tiles a workgroup, K shared (2560 x 10240: 4 rows (1, 4) 9.5 us, (4, 1) 22.3; 8 rows 11.8 and 23.8).  Some: (4, 1) (10240 x 2560: 4 rows 8.3, (1, 4)
// 10.4; 8 rows 8.7 and 14.1).  More rows than compute units take at once: whole rows, K shared only where it is long (51865 x 2560: 4 rows (2, 1) 22.1, (1, 4) 32; 8 rows 25.1 and
// 50; 20000 x 10240, 4 rows: (2, 4) 33.4, (2, 1) 35).
struct Q40Shape {
    int wr, wk;
};
static Q40Shape q40_shape(const Problem &p, int64_t tiles, const DeviceInfo &dev) {
    const int u = (int)((p.K + 511) / 512);
    const int64_t few = 2 * (int64_t)dev.num_cus, some = 4 * (int64_t)dev.num_cus;
    if (p.N > 16) {
        if (tiles <= few) return {2, p.K <= 1280 ? 2 : 4};
        return tiles <= some ? Q40Shape{4, 2} : Q40Shape{8, 1};
    }
    if (p.N > 8) {
        if (tiles <= few) return u <= 1 ? Q40Shape{4, 1} : Q40Shape{1, std::min(8, (int)((p.K + 255) / 256))};
        if (tiles <= some) return {4, u < 8 ? 1 : 2};
        const int64_t per = (tiles + dev.num_cus - 1) / dev.num_cus; // one workgroup per compute unit where it can have all of its rows
        return {per > 8 && per <= 16 ? (int)per : 8, 1};
    }
    if (tiles <= few) return u <= 1 ? Q40Shape{2, 1} : Q40Shape{1, std::min(u, u > 4 && u <= 8 ? 8 : 4)};
    if (tiles <= some) return {4, u < 8 ? 1 : 2};
    return {2, u < 8 ? 1 : u < 16 ? 2 : 4};
}

static hipError_t q40_run(const Problem &p, const void *A, const void *B, const void *bias, void *out, hipStream_t stream, const DeviceInfo &dev) {
    if (p.a_dt != RT_Q4_0 || p.act_dt != RT_F16 || p.N < 1 || p.b_ks != 1 || p.K < 128 || p.K % 32 != 0) return hipErrorNotSupported;
    if (p.stacks > 65535 || p.K > 1 << 22 || p.b_js > 1 << 23) return hipErrorNotSupported; // (offsets within a workgroup's rows in 32 bits)
    if (((uintptr_t)A & 15u) || ((uintptr_t)B & 15u) || (p.b_js * 2) % 16 || (p.b_bs * 2) % 16) return hipErrorNotSupported;
    GemvQ40Args g{};
    g.codes = (const uint8_t *)A;
    g.scales = (const half_t *)((const uint8_t *)A + q40_scale_offset((uint64_t)p.a_stack * p.M * p.K));
    g.X = (const half_t *)B, g.bias = (const half_t *)bias, g.out = (half_t *)out;
    g.M = p.M, g.N = p.N, g.K = p.K;
    g.a_stack = p.a_stack, g.b_stack = p.b_stack, g.b_bs = p.b_bs, g.b_js = p.b_js;
    g.o_bs = p.o_bs, g.o_is = p.o_is, g.o_js = p.o_js;
    g.has_bias = p.has_bias, g.bias_on_rows = p.bias_on_rows, g.act = p.act;
    g.vec_out = p.o_is == 1 && p.o_js % 8 == 0 && p.o_bs % 8 == 0 && ((uintptr_t)out & 15u) == 0;
    const Q40Shape c = q40_shape(p, (p.M + 15) / 16 * (p.N > 16 ? (p.N + 31) / 32 : 1) * p.stacks, dev);
    const int64_t st = p.stacks;
    if (p.N <= 4) {
        if (c.wr == 1) return launch_q40<1, 1, 4, 4, 1>(g, st, c.wr, c.wk, stream);
        if (c.wr == 2) return launch_q40<1, 1, 2, 4, 1>(g, st, c.wr, c.wk, stream);
        return launch_q40<1, 1, 1, 4, 1>(g, st, c.wr, c.wk, stream);
    }
    if (p.N <= 8) {
        if (c.wr == 1) return launch_q40<1, 2, 8, 4, 1>(g, st, c.wr, c.wk, stream);
        if (c.wr == 2) return launch_q40<1, 2, 4, 4, 1>(g, st, c.wr, c.wk, stream);
        return launch_q40<1, 2, 2, 4, 1>(g, st, c.wr, c.wk, stream);
    }
    if (p.N <= 16) {
        if (c.wr == 1) return launch_q40<1, 4, 8, 2, 2>(g, st, c.wr, c.wk, stream);
        if (c.wr == 4) return launch_q40<1, 4, 4, 4, 1>(g, st, c.wr, c.wk, stream);
        return launch_q40<1, 4, 2, 4, 1>(g, st, c.wr, c.wk, stream);
    }
    if (c.wr == 2) return launch_q40<2, 4, 8, 2, 1>(g, st, c.wr, c.wk, stream);
    if (c.wr == 4) return launch_q40<2, 4, 4, 2, 1>(g, st, c.wr, c.wk, stream);
    return launch_q40<2, 4, 2, 2, 1>(g, st, c.wr, c.wk, stream);
}

hipError_t launch_gemv_q40(const Problem &p, const void *A, const void *B, const void *bias, void *out, hipStream_t stream, const DeviceInfo &dev) {
    if (p.N > kGemvQ40MaxCols) return hipErrorNotSupported;
    const hipError_t e = launch_gemv_q40_rowdot(p, A, B, bias, out, stream, dev); // one or two vectors
    return e == hipErrorNotSupported ? q40_run(p, A, B, bias, out, stream, dev) : e;
}
// More rows: whole units of 256 of K against 160 weight rows and more are launch_gemm_nt's, but for what it leaves.  (Asked here too: a plan offers its product to
// the family that took it last time first, and whether that one takes it may go by the workspace.)
hipError_t launch_gemm_q40(const Problem &p, const void *A, const void *B, const void *bias, void *out, hipStream_t stream, const DeviceInfo &dev) {
    if (p.a_dt != RT_Q4_0 || (p.K % 256 == 0 && p.a_bs % 512 == 0 && p.M >= 160 && !gemm_nt_leaves_q4(p, dev))) return hipErrorNotSupported;
    return q40_run(p, A, B, bias, out, stream, dev);
}

} // namespace rt
