// Attention over a key/value cache held in 4-bit blocks (kernels_cache_q4.hip has the format), for one or a few query rows per head of keys:
//
//   out[m] = softmax_j(scale * sum_b dk[j, b] sum_{c in b} q[m, c] (qk[j, c] - 8) + mask[m, j]) . (dv[j, b] (qv[j, c] - 8))
//
// The rows m are the query rows of the heads that share a head of keys: m = query row * group + head of the group.
//
// A wavefront takes 64 keys at a time.  Scores: v_mfma_f32_16x16x32_f16 contracts a block of 32 for 16 rows and 16 keys, codes unscaled (exact), the
// block's sum scaled by dk in f32.  A load is 16 bytes a lane of consecutive pieces of consecutive keys, and a 4 x 4 transposition among lane
// groups puts dword g of a block into lane group g, as the operand wants it (kernels_gemv_q40.hip has the same step).  Rows up to 4 (8) are put at
// MFMA rows 4 m (4 m, 4 m + 1), where one result register (two) holds them all.
// Softmax: running reference and sum in f32; a row's keys are spread over 16 lanes, which four DPP rotations join for the maximum, and only at
// the end for the sum.
// Values: the operand of the second product holds, for one dimension, eight keys in a lane.  Codes of one key are neighbours along the dimensions, so
// lane c (of 16) reads four bytes of each key's row (two up to a head_dim of 64, one up to 32; a row of 80 takes ten lanes, which costs less than the second load
// that would occupy all), and a byte permutation of two keys' puts the same nibble of both into the two halves of a register: the unpacking of q40_codes with pairs of keys in place of pairs of dimensions.  The
// order of keys in that product is free: 4 r + s is key 16 s + r, so that a lane's four probabilities are neighbours.  dv (q - 8) is exact in f16 for
// scales of eight significant bits, which is what the cache's write makes (others round here); dv = 0 past the last key.  The probabilities enter as
// f16, as in kernels_attention.hip.
//
// Wavefronts of a workgroup take 64 keys in turn and are merged through LDS; where there are few heads several workgroups share the keys and a second
// kernel merges them, in a fixed order.
//
// 32 sequences of 8192 keys, 8 heads of 128, one row of 32 heads: 60 us from HBM, 5.0 TB/s, near a copy's 5.1 (53 over and over on one state, of which the last-level cache
// keeps some); of lengths between, whose longest bounds it, 51 (46).  Small ones wait: 32768 keys of one sequence 16.0 us from HBM, 14.3 on one state (7.4 at a copy's rate), in a
// launch, a trip to memory and two steps of 1.7 us in which two wavefronts of a SIMD unpack (500 instructions for 64 keys), and 3 of the second launch.
#include "device_common.h"

#include <algorithm>
#include <cmath>

namespace rt {

constexpr float kLog2eQ4 = 1.4426950408889634f;
constexpr int AQ_MAX_SPLITS = 64; // shares of a row of the prompt kernel
constexpr int AQ_WAVES = 8;       // of a streaming workgroup
// The exponentials' reference (mx, m_run below) is this much, in base 2, below a block's maximum.  As f16 a probability goes down to 2^-25, so that against the largest none of
// more than 2^-32 is lost (with the maximum itself as reference 2^16 keys of 2^-25.5 each beside one of 1 were, an eighth or half of them, those of its wavefront).  Below 8, since
// what is left of a difference of 8 and more may round to 16 where an f32's step is that, between 2^27 and 2^28, and 2^16 is no f16.
constexpr float AQ_BELOW = 7.f;

struct AttnQ4Args {
    const half_t *Q;
    const uint8_t *Kc, *Vc;
    const half_t *Ks, *Vs;
    const void *mask;
    const int32_t *lens;
    half_t *O;
    float *part_o, *part_ml; // [row][split][D], [row][split][2]
    int64_t q_bs, q_hs, q_rs, o_bs, o_hs, o_rs, m_bs, m_rs;
    int kv_heads, group, rows, kv_len, q_len, capacity; // rows = q_len * group
    int causal, mask_f32, splits, split_keys, row_tiles;
    float scale, scale_log2e;
};

// Scores and references are in units of log2(e), and with a mask tensor as they are, in the kernels and in the partial results: f32's lowest number, which hides nothing from a row
// that has nothing else, and its neighbours would be infinite in the others.
__host__ __device__ constexpr float aq_unit(bool masked) { return masked ? kLog2eQ4 : 1.f; }

template <int CTRL> __device__ __forceinline__ float aq_dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float aq_max16(float v) {
    v = fmaxf(v, aq_dpp<0x128>(v)), v = fmaxf(v, aq_dpp<0x124>(v));
    v = fmaxf(v, aq_dpp<0x122>(v));
    return fmaxf(v, aq_dpp<0x121>(v));
}
__device__ __forceinline__ float aq_sum16(float v) {
    v += aq_dpp<0x128>(v), v += aq_dpp<0x124>(v);
    v += aq_dpp<0x122>(v);
    return v + aq_dpp<0x121>(v);
}
__device__ __forceinline__ uint32_t aq_or16(uint32_t v) {
    v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true);
    v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true);
    v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true);
    return v | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true);
}

// How a row of values, 8 NT bytes, is read by 16 lanes: W bytes each, by CL of them
template <int NT> struct AqDims {
    static constexpr int D = 16 * NT, RB = 8 * NT, NF = D / 32, TAIL = NT & 1, NB = NF + TAIL, SR = NB == 3 ? 4 : NB, PB = NF ? NF : 1; // (PB: pieces of 16 bytes of a key, where there are any)
    static constexpr int W = NT > 4 ? 4 : NT > 2 ? 2 : 1, CL = RB / W, T = 2 * W;
    // dimension that lane c's column of tile t stands for
    __device__ __forceinline__ static int dim(int t, int c) {
        const int nibble = T * c + t; // of the row
        return 8 * (nibble >> 3) + ((nibble & 3) << 1) + ((nibble >> 2) & 1);
    }
};

// Whether the f16 values of a scale are finite: eight times 8188 is 65504, the largest.  One past it (the cache's write makes none) counts as one that is not finite: as
// an infinite operand of the matrix cores, a key that a row does not see would reach it as 0 * inf.
__device__ __forceinline__ bool aq_finite(uint32_t bits) { return (bits & 0x7FFFu) <= 0x6FFFu; }

// Loads with a bound: past `bytes` the hardware returns zeros, and so codes of keys past the last have scales of zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t aq_bounded(const void *p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00027000); // raw, 32-bit data
}

// VPR: result registers in use (1: up to 4 rows, 2: up to 8, 4: up to 16).  MK: a mask tensor
template <int NT, int VPR, int MK> __global__ __launch_bounds__(512) void attention_q4_kernel(AttnQ4Args g) {
    using DM = AqDims<NT>;
    constexpr int D = DM::D, NF = DM::NF, TAIL = DM::TAIL, NB = DM::NB, SR = DM::SR, SW = (SR + 1) / 2, RB = DM::RB, W = DM::W, T = DM::T;
    constexpr int ROWS = 4 * VPR, PS = 72; // halves between rows of probabilities
    constexpr int WAVE_LDS = (ROWS * PS + NB * 64) * 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int waves = AQ_WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, fg = lane >> 4, cc = min(r, DM::CL - 1);
    half_t *P = (half_t *)(smem + wave * WAVE_LDS), *S = P + ROWS * PS; // this wavefront's: probabilities [row][position], scales of values [block][position]
    const int bk = blockIdx.y, b = bk / g.kv_heads, kh = bk - b * g.kv_heads;

    int len = g.kv_len;
    if (g.lens) len = min(max(g.lens[b], 0), len);
    // row fg VPR + v: its query row, head and last visible key
    auto q_row = [&](int m) { return min(m, g.rows - 1) / g.group; };
    int last[VPR];
#pragma unroll
    for (int v = 0; v < VPR; v++) last[v] = g.causal ? min(len - 1, q_row(fg * VPR + v) + len - g.q_len) : len - 1;
    // the keys of this workgroup: its share of those that any row sees; up to `whole` all rows see them all
    const int end = g.causal ? min(len, q_row(g.rows - 1) + len - g.q_len + 1) : len, whole = g.causal ? min(len, len - g.q_len + 1) : len;
    const int j_first = blockIdx.x * g.split_keys;
    const int j_end = min(end, j_first + g.split_keys);

    const int64_t head = (int64_t)bk * g.capacity;
    const uint8_t *const Kc = g.Kc + head * RB, *const Vc = g.Vc + head * RB;
    const half_t *const Ks = g.Ks + head * SR, *const Vs = g.Vs + head * SR;

    half8_t qf[NB];
    {
        const int m = min((r >> 2) * VPR + min(r & 3, VPR - 1), g.rows - 1), qi = m / g.group;
        const half_t *q = g.Q + b * g.q_bs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.q_hs + qi * g.q_rs + 8 * fg;
#pragma unroll
        for (int k = 0; k < NF; k++) qf[k] = *(const half8_t *)(q + 32 * k);
        if constexpr (TAIL) qf[NF] = fg < 2 ? *(const half8_t *)(q + 32 * NF) : half8_t{};
    }

    // ---- 64 keys' loads, the wavefront's next
    const int step = 64 * waves;
    struct Unit {
        uint4_t kc[NF + TAIL];
        uint32_t dk[SW], dv[SW]; // lane group fg has the scales of keys 16 fg + r
        uint32_t v[2][8];
    };
    // offsets of this lane's loads in 32 bits from the first key of a window of 2^24: pieces of 16 bytes of keys (a constant apart but where a key has three), a
    // block of 16, scales, values
    uint32_t ko[DM::PB == 3 ? 3 : 1], kt, so, vo;
    __amdgpu_buffer_rsrc_t kr, vr, ksr, vsr;
    auto window = [&](int j0, int j1) __attribute__((always_inline)) { // the keys j0 .. j1 - 1; this wavefront's start 64 wave behind
#pragma unroll
        for (int i = 0; i < (DM::PB == 3 ? 3 : 1); i++) {
            const int pc = 4 * i + fg, ks = pc / DM::PB, kb = pc - ks * DM::PB; // piece: key set and block
            ko[i] = (64 * wave + 16 * ks + r) * RB + 16 * kb;
        }
        kt = (64 * wave + lane) * RB + 16 * NF, so = (64 * wave + lane) * SR * 2, vo = (64 * wave + 2 * fg) * RB + W * cc;
        kr = aq_bounded(Kc + (int64_t)j0 * RB, (j1 - j0) * RB), vr = aq_bounded(Vc + (int64_t)j0 * RB, (j1 - j0) * RB);
        ksr = aq_bounded(Ks + (int64_t)j0 * SR, (j1 - j0) * SR * 2), vsr = aq_bounded(Vs + (int64_t)j0 * SR, (j1 - j0) * SR * 2);
    };
    auto load = [&](Unit &k) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NF; i++)
            k.kc[i] = __builtin_bit_cast(uint4_t, DM::PB == 3 ? __builtin_amdgcn_raw_buffer_load_b128(kr, ko[i], 0, 0) : __builtin_amdgcn_raw_buffer_load_b128(kr, ko[0] + i * (64 / DM::PB) * RB, 0, 0));
        if constexpr (TAIL) {
            const uint2_t w = __builtin_bit_cast(uint2_t, __builtin_amdgcn_raw_buffer_load_b64(kr, kt, 0, 0));
            k.kc[NF] = uint4_t{w[0], w[1], 0, 0};
        }
        auto scales = [&](__amdgpu_buffer_rsrc_t p, uint32_t *d) __attribute__((always_inline)) {
            if constexpr (SR == 1) d[0] = __builtin_amdgcn_raw_buffer_load_b16(p, so, 0, 0);
            else if constexpr (SR == 2) d[0] = __builtin_amdgcn_raw_buffer_load_b32(p, so, 0, 0);
            else {
                const uint2_t x = __builtin_bit_cast(uint2_t, __builtin_amdgcn_raw_buffer_load_b64(p, so, 0, 0));
                d[0] = x[0], d[SW - 1] = x[1];
            }
        };
        scales(ksr, k.dk), scales(vsr, k.dv);
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t o = vo + (16 * (e & 3) + 8 * u + (e >> 2)) * RB;
                if constexpr (W == 4) k.v[u][e] = __builtin_amdgcn_raw_buffer_load_b32(vr, o, 0, 0);
                else if constexpr (W == 2) k.v[u][e] = __builtin_amdgcn_raw_buffer_load_b16(vr, o, 0, 0);
                else k.v[u][e] = __builtin_amdgcn_raw_buffer_load_b8(vr, o, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < (DM::PB == 3 ? 3 : 1); i++) ko[i] += step * RB;
        kt += step * RB, so += step * SR * 2, vo += step * RB;
    };
    uint32_t mk[MK ? VPR : 1][4]; // the block's mask values, as they are; requested before the next block's loads, so that nothing waits for those
    auto load_mask = [&](int j0) __attribute__((always_inline)) {
        if constexpr (MK != 0) {
#pragma unroll
            for (int v = 0; v < VPR; v++) {
                const int64_t row = b * g.m_bs + q_row(fg * VPR + v) * g.m_rs;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const int64_t i = row + min(j0 + 16 * s + r, len - 1);
                    mk[v][s] = g.mask_f32 ? ((const uint32_t *)g.mask)[i] : ((const uint16_t *)g.mask)[i];
                }
            }
        }
    };

    constexpr float unit = aq_unit(MK);
    float mx[VPR], sum[VPR];
    uint32_t bad[VPR];
    float4_t o[T];
#pragma unroll
    for (int v = 0; v < VPR; v++) mx[v] = -INFINITY, sum[v] = 0.f, bad[v] = 0;
#pragma unroll
    for (int n = 0; n < T; n++) o[n] = float4_t{0.f, 0.f, 0.f, 0.f};
    const uint32_t bias = q40_bias();

    auto multiply = [&](int j0, Unit &k) __attribute__((always_inline)) {
        // ---- scores
        uint32_t dk[SW][4]; // of key 16 s + r
#pragma unroll
        for (int w = 0; w < SW; w++) q40_spread<4>(k.dk[w], dk[w]);
        float sc[4][VPR];
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int v = 0; v < VPR; v++) sc[s][v] = 0.f;
        // a block's sums are folded behind the next block's instructions: left alone the compiler waits for the matrix cores after each
        float4_t part = {0.f, 0.f, 0.f, 0.f};
        float scale = 0.f;
        int set = 0;
        auto fold = [&]() __attribute__((always_inline)) {
            asm volatile("" : "+v"(part));
#pragma unroll
            for (int v = 0; v < VPR; v++) sc[set][v] = fmaf(scale, part[v], sc[set][v]);
        };
        auto block = [&](uint32_t w, int s, int n) __attribute__((always_inline)) {
            const float4_t now = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[n], q40_codes(w, bias), float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            fold();
            part = now, scale = (float)__builtin_bit_cast(half2_t, dk[n >> 1][s])[n & 1], set = s;
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int i = 0; i < NF; i++) {
            q40_transpose(k.kc[i]);
#pragma unroll
            for (int x = 0; x < 4; x++) block(k.kc[i][x], (4 * i + x) / DM::PB, (4 * i + x) % DM::PB);
        }
        if constexpr (TAIL) {
            q40_transpose(k.kc[NF]);
#pragma unroll
            for (int s = 0; s < 4; s++) block(k.kc[NF][s], s, NF);
        }
        fold();

        // ---- mask, running maximum and sum, probabilities to LDS
        const bool inside = j0 + 64 <= whole; // no key hidden
#pragma unroll
        for (int v = 0; v < VPR; v++) {
#pragma unroll
            for (int s = 0; s < 4; s++) {
                float x;
                if constexpr (MK != 0) {
                    const float mv = g.mask_f32 ? __builtin_bit_cast(float, mk[v][s]) : (float)__builtin_bit_cast(half_t, (uint16_t)mk[v][s]);
                    x = mv == -INFINITY ? -INFINITY : fmaf(sc[s][v], g.scale, mv); // (a hidden key's score may be anything)
                } else {
                    x = sc[s][v] * g.scale_log2e;
                }
                if (!inside) x = j0 + 16 * s + r <= last[v] ? x : -INFINITY;
                sc[s][v] = x;
            }
            const float top = fmaxf(mx[v], aq_max16(fmaxf(fmaxf(sc[0][v], sc[1][v]), fmaxf(sc[2][v], sc[3][v]))) - AQ_BELOW / unit);
            const float base = top == -INFINITY ? 0.f : top;
            const float a = __builtin_amdgcn_exp2f((mx[v] - base) * unit);
            mx[v] = top;
            float l = 0.f;
            half4_t p4;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float p = __builtin_amdgcn_exp2f((sc[s][v] - base) * unit);
                p4[s] = (half_t)p;
                if (MK == 0) l += p;
            }
            // In base 2 the largest probability is a power of two, as f16 too.  In other units it is one only where a score's step is small beside 1: the sum is that of the rounded
            // probabilities there, so that what the largest, or equal ones, lose is in both.
            if constexpr (MK != 0) {
                const half2_t one = {(half_t)1, (half_t)1};
                l = __builtin_amdgcn_fdot2(half2_t{p4[2], p4[3]}, one, __builtin_amdgcn_fdot2(half2_t{p4[0], p4[1]}, one, 0.f, false), false);
            }
            sum[v] = fmaf(sum[v], a, l);
#pragma unroll
            for (int n = 0; n < T; n++) o[n][v] *= a;
            *(half4_t *)(P + (fg * VPR + v) * PS + 4 * r) = p4;
        }
        // ---- scales of the values to LDS; one that is not finite shows in the rows that see its key and not through the matrix cores
        uint32_t odd = 0;
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const half_t d = __builtin_bit_cast(half2_t, k.dv[n >> 1])[n & 1];
            const bool fin = aq_finite(__builtin_bit_cast(uint16_t, d));
            if (!fin) odd |= 1u << n;
            S[n * 64 + 4 * r + fg] = fin ? d : (half_t)0.f;
        }
        if (__builtin_amdgcn_ballot_w64(odd != 0)) {
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const uint32_t ks = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (16 * s + r), (int)odd);
#pragma unroll
                for (int v = 0; v < VPR; v++)
                    if (!(sc[s][v] == -INFINITY)) bad[v] |= ks;
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");

        // ---- values
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const half8_t pf = *(const half8_t *)(P + ((r >> 2) * VPR + min(r & 3, VPR - 1)) * PS + 32 * u + 8 * fg);
            const half8_t d = *(const half8_t *)(S + ((T * cc) >> 5) * 64 + 32 * u + 8 * fg);
            // four registers of key pairs: nibble `n` of the halves -> operand of tile `n0 + n`
            auto product = [&](const uint32_t *w, int n0, int count) __attribute__((always_inline)) {
                half8_t c[4];
#pragma unroll
                for (int e = 0; e < 4; e++) c[e] = q40_codes(w[e], bias);
#pragma unroll
                for (int n = 0; n < count; n++) {
                    const half8_t x = half8_t{c[0][2 * n], c[0][2 * n + 1], c[1][2 * n], c[1][2 * n + 1], c[2][2 * n], c[2][2 * n + 1], c[3][2 * n], c[3][2 * n + 1]} * d;
                    o[n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, x, o[n0 + n], 0, 0, 0);
                }
            };
            uint32_t w[4];
            if constexpr (W == 4) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = __builtin_amdgcn_perm(k.v[u][2 * e + 1], k.v[u][2 * e], hf ? 0x07060302u : 0x05040100u);
                    product(w, 4 * hf, 4);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = k.v[u][2 * e] | (k.v[u][2 * e + 1] << 16);
                product(w, 0, T);
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
    };

    // 64 keys are multiplied while the wavefront's next 64 are on their way
    constexpr int WINDOW = 1 << 24;
    Unit ring[2];
#pragma unroll 1
    for (int w0 = j_first; w0 < j_end; w0 += WINDOW) {
        const int w1 = min(j_end - w0, WINDOW) + w0;
        window(w0, w1);
        int j0 = w0 + 64 * wave;
        load(ring[0]);
        __builtin_amdgcn_sched_barrier(0);
        auto turn = [&](int j, Unit &now, Unit &next) __attribute__((always_inline)) {
            load_mask(j);
            load(next); // (past the end: zeros)
            __builtin_amdgcn_sched_barrier(0);
            multiply(j, now);
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll 1
        for (; j0 + step < w1; j0 += 2 * step) {
            turn(j0, ring[0], ring[1]);
            turn(j0 + step, ring[1], ring[0]);
        }
        if (j0 < w1) load_mask(j0), multiply(j0, ring[0]);
    }

    // ---- this wavefront's rows: the sum over the 16 lanes, and what a scale that is not finite leaves
#pragma unroll
    for (int v = 0; v < VPR; v++) {
        sum[v] = aq_sum16(sum[v]);
        const uint32_t bd = aq_or16(bad[v]);
#pragma unroll
        for (int n = 0; n < T; n++)
            if ((bd >> (DM::dim(n, cc) >> 5)) & 1u) o[n][v] = __builtin_nanf("");
    }
    // ---- the wavefronts' results through LDS: outputs [wave][T][VPR][64], maxima and sums [wave][row][2]
    constexpr int PER = T * VPR * 64;
    float *red = (float *)smem, *ml = red + waves * PER;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < T; n++)
#pragma unroll
        for (int v = 0; v < VPR; v++) red[wave * PER + (n * VPR + v) * 64 + lane] = o[n][v];
#pragma unroll
    for (int v = 0; v < VPR; v++) {
        const int row = fg * VPR + v;
        if (r == 0) ml[(wave * ROWS + row) * 2] = mx[v], ml[(wave * ROWS + row) * 2 + 1] = sum[v];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < PER; e += blockDim.x) {
        const int l = e & 63, v = (e >> 6) % VPR, n = (e >> 6) / VPR, m = (l >> 4) * VPR + v;
        if (m >= g.rows || (l & 15) >= DM::CL) continue;
        float top = -INFINITY;
        for (int w = 0; w < waves; w++) top = fmaxf(top, ml[(w * ROWS + m) * 2]);
        const float base = top == -INFINITY ? 0.f : top;
        float y = 0.f, s = 0.f;
        for (int w = 0; w < waves; w++) {
            const float a = __builtin_amdgcn_exp2f((ml[(w * ROWS + m) * 2] - base) * unit);
            y = fmaf(red[w * PER + e], a, y), s = fmaf(ml[(w * ROWS + m) * 2 + 1], a, s);
        }
        const int d = DM::dim(n, l & 15);
        if (g.splits > 1) {
            const int64_t at = ((int64_t)bk * g.rows + m) * g.splits + blockIdx.x;
            g.part_o[at * D + d] = y;
            if (d == 0) g.part_ml[2 * at] = top, g.part_ml[2 * at + 1] = s;
        } else {
            const int qi = m / g.group;
            g.O[b * g.o_bs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.o_hs + qi * g.o_rs + d] = (half_t)(y / s); // no visible key: 0 / 0
        }
    }
}

// ---------------------------------------------------------------------------------------------
// More rows (prompts, and steps of a few tokens with heads that share keys): a workgroup of four wavefronts has 128 rows of one head of keys, a wavefront 32 of
// them, against blocks of 64 keys that all four widen to f16 in LDS: d (q - 8), which is exact for scales of eight significant bits, as the cache's write makes
// them (others round here).  Widening costs 15 instructions for eight values, once for 128 rows; the kernel above does it for every 16.  A thread's share of
// the next block (a dword of codes per 16 dimensions) is requested before this block's products and widened behind them, into the other of two stages.
// LDS rows are 16 bytes longer than the values: the fragments' reads then meet no bank twice.
//   S = K Q^T: keys first, so that a lane holds one row's scores of 16 keys, and the maximum needs two steps across lanes.
//   O += V^T P: the lane's probabilities are an operand as they lie; the values' comes transposed out of LDS (ds_read_b64_tr_b16).
// The exponentials' reference follows the row's maximum only where that has risen by some 2^8, so that outputs and sums are seldom rescaled; f16 rounds a probability
// of 2^15 as it does one of 1, relatively.  The sum is that of the rounded probabilities.
// Two groups of four wavefronts have halves of the 128 keys of a step and are joined at the end: one workgroup per compute unit then has two wavefronts per SIMD at any
// length (four wavefronts and two workgroups took as long as the longer of the two: 2048 x 2048 x 32 heads x 96 causal 70 us, this 50).
// us: 2048 x 2048 x 32 heads, causal, of 96 / 128 dimensions 50 / 59; 2 x 512 rows of 32 heads on 8 x 4096 keys of 128 87 (790 TFLOP/s), of 64 59.  Bound by instruction
// issue: softmax and widening take 48 % of the cycles, the MFMAs 22 % beside them.
// ---------------------------------------------------------------------------------------------
constexpr int AP_ROWS = 128, AP_KEYS = 128; // of a workgroup's step
typedef half_t half4_u __attribute__((ext_vector_type(4), aligned(2))); // outputs start anywhere
typedef __fp16 aq_fp16x4 __attribute__((ext_vector_type(4)));

// halves of a row of values in LDS, of a stage
constexpr int aq_value_row(int nt) { return 16 * nt + (nt % 2 ? 0 : 16); }
constexpr int aq_stage(int nt) { return AP_KEYS * (16 * nt + 8 + aq_value_row(nt)); }

// MK: no mask tensor, an f32 one, an f16 one
template <int NT, int MK> __global__ __launch_bounds__(512, 2) void attention_q4_tile_kernel(AttnQ4Args g) {
    constexpr int D = 16 * NT, KK = (NT + 1) / 2, RB = D / 2, SR = KK == 3 ? 4 : KK, DW = 2 * NT;            // (DW: dwords of a row)
    constexpr int LD = D + 8, VD = aq_value_row(NT), KBLK = AP_KEYS * LD, STAGE = aq_stage(NT); // halves: a row of keys, of values; a block of keys, both
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    half_t *const ring = (half_t *)smem;                          // [2][keys | values][128][LD | VD]
    uint32_t *const odd_flags = (uint32_t *)(ring + 2 * STAGE);   // [2][wavefront]: whether the block has a scale of values, of keys that is not finite
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int fr = lane & 15, fg = lane >> 4, rg = wave & 3, kg = wave >> 2; // group of rows, half of the keys

    // (head of keys, tile of rows, share of keys): XCD x takes the x-th eighth, so that a head's tiles share an L2; with the causal flag the long (late) tiles
    // come first
    uint32_t lin = blockIdx.x, bk, tile, sp = 0;
    const uint32_t total = gridDim.x, nt = (uint32_t)g.row_tiles;
    const uint32_t chunk = total >> 3, rr = lin >> 3, x8 = lin & 7u;
    if ((total & 7u) == 0 && g.causal && g.splits == 1 && chunk % nt == 0) {
        const uint32_t hx = chunk / nt, q = rr / hx;
        bk = x8 * hx + (rr - q * hx);
        tile = nt - 1 - q;
    } else {
        if ((total & 7u) == 0) lin = x8 * chunk + rr;
        const uint32_t u = lin / (uint32_t)g.splits;
        sp = lin - u * (uint32_t)g.splits;
        bk = u / nt, tile = u - bk * nt;
    }
    const int b = (int)bk / g.kv_heads, kh = (int)bk - b * g.kv_heads;
    const int row0 = (int)tile * AP_ROWS, rw = row0 + 32 * rg; // first row of the workgroup, of the wavefront
    int len = g.kv_len;
    if (g.lens) len = min(max(__builtin_amdgcn_readfirstlane(g.lens[b]), 0), len);
    const int off = len - g.q_len; // causal: query row i sees keys <= i + off
    auto sees = [&](int m) { return g.causal ? max(0, min(len, min(m, g.rows - 1) / g.group + off + 1)) : len; }; // keys that row m sees
    const int j_first = (int)sp * g.split_keys;
    const int j_end = min(sees(row0 + AP_ROWS - 1), j_first + g.split_keys), w_end = rw < g.rows ? min(j_end, sees(rw + 31)) : 0;
    const int w_lean = MK || g.scale_log2e > 0.f ? min(w_end, sees(rw)) : 0; // blocks up to here: every key is seen by all of the wavefront's rows

    const int64_t head = (int64_t)bk * g.capacity;
    const uint8_t *const Kc = g.Kc + head * RB, *const Vc = g.Vc + head * RB;
    const half_t *const Ks = g.Ks + head * SR, *const Vs = g.Vs + head * SR;

    // rows rw + 16 u + fr: fragments of dimensions 32 kk + 8 fg .. + 7 (zero past head_dim)
    half8_t fq[2][KK];
    int last[2]; // the last key that the row sees
    bool wild = false; // whether a query that is not finite is among them
    const half_t *mrow[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int m = min(rw + 16 * u + fr, g.rows - 1), qi = m / g.group;
        last[u] = (g.causal ? min(len, qi + off + 1) : len) - 1;
        const half_t *qp = g.Q + b * g.q_bs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.q_hs + qi * g.q_rs;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) fq[u][kk] = 32 * kk + 8 * fg < D ? *(const half8_t *)(qp + 32 * kk + 8 * fg) : half8_t{};
        if (MK)
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int e = 0; e < 8; e++) wild |= !(__builtin_fabsf((float)fq[u][kk][e]) <= 65504.f);
        mrow[u] = (const half_t *)g.mask + (b * g.m_bs + qi * g.m_rs) * (MK == 1 ? 2 : 1);
    }

    wild = __builtin_amdgcn_ballot_w64(wild) != 0;
    // awaited here: a first use in the loop, where the compiler does not know them from the block's loads, waited for those in every step
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int kk = 0; kk < KK; kk++) asm volatile("" : "+v"(fq[u][kk]));
    // ---- this thread's dwords of a block: number i is dword i * 512 + t of [keys | values][128][DW], at four times that from the block's first
    uint32_t raw[NT], ds[NT], so[NT]; // (so: of its scale; the key is so / (2 SR))
    auto is_key = [&](int i) { return 2 * i + 2 <= NT || (2 * i < NT && wave < 4); }; // (uniform)
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int f = (i * 512 + t) % (256 * NT), key = f / DW;
        so[i] = 2 * (key * SR + ((f - key * DW) >> 2));
    }
    auto load = [&](int j) __attribute__((always_inline)) {
        const int j0 = __builtin_amdgcn_readfirstlane(j), n = min(AP_KEYS, len - j0); // past the last key the loads return zeros
        const auto kr = aq_bounded(Kc + (int64_t)j0 * RB, n * RB), vr = aq_bounded(Vc + (int64_t)j0 * RB, n * RB);
        const auto ksr = aq_bounded(Ks + (int64_t)j0 * SR, n * SR * 2), vsr = aq_bounded(Vs + (int64_t)j0 * SR, n * SR * 2);
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int e = i * 512 + t;
            if (is_key(i)) {
                raw[i] = __builtin_amdgcn_raw_buffer_load_b32(kr, 4 * e, 0, 0), ds[i] = __builtin_amdgcn_raw_buffer_load_b16(ksr, so[i], 0, 0);
            } else {
                raw[i] = __builtin_amdgcn_raw_buffer_load_b32(vr, 4 * e - 1024 * NT, 0, 0), ds[i] = __builtin_amdgcn_raw_buffer_load_b16(vsr, so[i], 0, 0);
            }
        }
    };
    const uint32_t bias = q40_bias();
    auto widen = [&](int stage) __attribute__((always_inline)) {
        uint8_t *const st = (uint8_t *)(ring + stage * STAGE);
        bool odd = false, odd_key = false;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const bool val = !is_key(i);
            const uint32_t f = (uint32_t)(i * 512 + t - (val ? 256 * NT : 0)), key = so[i] / (2 * SR);
            half_t d = __builtin_bit_cast(half_t, (uint16_t)ds[i]);
            const bool fin = aq_finite(ds[i]);
            if (val) { // a value that is not finite shows in the rows that see its key, and not through the matrix cores
                odd |= !fin;
                d = fin ? d : (half_t)0.f;
            } else if (MK) {
                odd_key |= !fin;
            }
            *(half8_t *)(st + 16 * f + (val ? 2 * KBLK + (VD - D) * 2 * key : (LD - D) * 2 * key)) = q40_codes(raw[i], bias) * half8_t{d, d, d, d, d, d, d, d};
        }
        const uint32_t any = (__builtin_amdgcn_ballot_w64(odd) != 0 ? 1u : 0u) | (__builtin_amdgcn_ballot_w64(odd_key) != 0 ? 2u : 0u);
        if (lane == 0) odd_flags[8 * stage + wave] = any;
    };
    using MT = std::conditional_t<MK == 1, float, half_t>;
    typedef MT mask4_t __attribute__((ext_vector_type(4)));
    typedef MT mask4_u __attribute__((ext_vector_type(4), aligned(sizeof(MT)))); // rows start anywhere
    constexpr int MU = MK ? 2 : 1, MB = MK ? 4 : 1;
    mask4_t mk[MU][MB]; // the wavefront's next block's, requested before the second product of the one before it
    auto load_mask = [&](int j0) __attribute__((always_inline)) {
        if constexpr (MK != 0) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const MT *p = (const MT *)mrow[u];
                if (j0 + 64 <= len) { // uniform
#pragma unroll
                    for (int bt = 0; bt < 4; bt++) mk[u][bt] = *(const mask4_u *)(p + j0 + 16 * bt + 4 * fg);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) mk[u][e >> 2][e & 3] = p[min(j0 + 16 * (e >> 2) + 4 * fg + (e & 3), len - 1)];
                }
            }
        }
    };

    float4_t acc[2][NT];
    // the exponentials' reference and this lane's share of the sum
    constexpr float unit = aq_unit(MK);
    float m_run[2], l_run[2];
    uint32_t bad[2];
    bool coarse = false; // whether a reference was too large for scores that are not rounded (uniform)
#pragma unroll
    for (int u = 0; u < 2; u++) {
        m_run[u] = -INFINITY, l_run[u] = 0.f, bad[u] = 0;
#pragma unroll
        for (int d = 0; d < NT; d++) acc[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    int koff[KK];
#pragma unroll
    for (int kk = 0; kk < KK; kk++) koff[kk] = (64 * kg + fr) * LD + 8 * min(4 * kk + fg, DW - 1);
    const int voff = KBLK + (64 * kg + 4 * fg + (fr >> 2)) * VD + 4 * (fr & 3);

    auto step = [&](int stage, int j0, auto lean_c) __attribute__((always_inline)) {
        constexpr bool LEAN = decltype(lean_c)::value;
        const half_t *const st = ring + stage * STAGE;
        const uint4_t fl = *(const uint4_t *)(odd_flags + 8 * stage), fh = *(const uint4_t *)(odd_flags + 8 * stage + 4);
        float4_t S[2][4];
#pragma unroll
        for (int bt = 0; bt < 4; bt++) {
            half8_t fk[KK];
#pragma unroll
            for (int kk = 0; kk < KK; kk++) fk[kk] = *(const half8_t *)(st + koff[kk] + 16 * bt * LD);
#pragma unroll
            for (int u = 0; u < 2; u++) S[u][bt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int u = 0; u < 2; u++) S[u][bt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fk[kk], fq[u][kk], S[u][bt], 0, 0, 0);
        }
        const uint32_t flags = (uint32_t)__builtin_amdgcn_readfirstlane((int)(fl[0] | fl[1] | fl[2] | fl[3] | fh[0] | fh[1] | fh[2] | fh[3]));
        const bool odd = flags & 1u;
        half8_t fp[2][2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float bmax = -INFINITY;
            if constexpr (LEAN && MK == 0) { // scale > 0: the maximum of the raw scores, the scale folded into the exponent's argument
#pragma unroll
                for (int e = 0; e < 16; e++) bmax = fmaxf(bmax, S[u][e >> 2][e & 3]);
                bmax *= g.scale_log2e;
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float s = S[u][e >> 2][e & 3];
                    S[u][e >> 2][e & 3] = MK ? fmaf(s, g.scale, (float)mk[MK ? u : 0][MK ? e >> 2 : 0][e & 3]) : s * g.scale_log2e;
                }
                if (MK && ((flags & 2u) || wild)) { // a hidden key's score may be anything
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if ((float)mk[MK ? u : 0][MK ? e >> 2 : 0][e & 3] == -INFINITY) S[u][e >> 2][e & 3] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    if (!LEAN && j0 + 16 * (e >> 2) + 4 * fg + (e & 3) > last[u]) S[u][e >> 2][e & 3] = -INFINITY;
                    bmax = fmaxf(bmax, S[u][e >> 2][e & 3]);
                }
            }
            if (odd) {
                uint32_t seen = 0;
#pragma unroll
                for (int e = 0; e < 16; e++) seen |= S[u][e >> 2][e & 3] == -INFINITY ? 0u : 1u << e;
#pragma unroll 1
                for (int e = 0; e < 16 * KK; e++) {
                    const int k = e >> 4;
                    const uint32_t j = (uint32_t)min(j0 + 4 * (e & 12) + 4 * fg + (e & 3), len - 1);
                    const bool fin = aq_finite(__builtin_bit_cast(uint16_t, Vs[j * SR + k]));
                    if (!fin && ((seen >> (e & 15)) & 1u)) bad[u] |= 1u << k;
                }
            }
            bmax = rt_groups_max(bmax);
            // the reference follows the maximum only where that is some 2^15 past it (or it has none), and then 2^8 past where it was: the outputs and the sum are seldom rescaled.
            // (Their difference, which is exact where it is small: a sum may round.  2^15 is below f16's last, 2^16 is not.)
            float sc = LEAN && MK == 0 ? g.scale_log2e : 1.f;
            if (__builtin_amdgcn_ballot_w64(bmax - m_run[u] > 15.f / unit)) {
                const float m_new = fmaxf(m_run[u], bmax - AQ_BELOW / unit), alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run[u] - m_new) * unit);
                m_run[u] = m_new;
                l_run[u] *= alpha;
#pragma unroll
                for (int d = 0; d < NT; d++) acc[u][d] *= alpha;
                // The reference is a rounded product and a score meets it in the fused multiply-add without a rounding of its own: past 4096 that shows, 2^-12 and more between
                // blocks here and those that round their scores, and past 2^28 a probability would leave f16.  From there on scores are rounded first.
                if (LEAN && MK == 0 && __builtin_amdgcn_ballot_w64(!(__builtin_fabsf(m_new) < 4096.f))) {
                    coarse = true;
#pragma unroll
                    for (int e = 0; e < 16; e++) S[u][e >> 2][e & 3] *= g.scale_log2e;
                    sc = 1.f;
                }
            }
            const float m_use = m_run[u] == -INFINITY ? 0.f : m_run[u]; // a row without a key yet: exp2(-inf - 0) = 0
            float psum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float s0 = S[u][e >> 2][e & 3], s1 = S[u][e >> 2][(e & 3) + 1];
                const float p0 = __builtin_amdgcn_exp2f(MK ? (s0 - m_use) * unit : fmaf(s0, sc, -m_use)), p1 = __builtin_amdgcn_exp2f(MK ? (s1 - m_use) * unit : fmaf(s1, sc, -m_use));
                const half2_t p = {(half_t)p0, (half_t)p1};
                psum = __builtin_amdgcn_fdot2(p, half2_t{(half_t)1, (half_t)1}, psum, false);
                fp[u][e >> 3][e & 7] = p[0], fp[u][e >> 3][(e & 7) + 1] = p[1];
            }
            l_run[u] += psum;
        }
        load_mask(j0 + AP_KEYS); // in registers that are free from here on
#pragma unroll
        for (int hh = 0; hh < 2; hh++)
#pragma unroll
            for (int d = 0; d < NT; d++) {
                typedef uint64_t u64x2_t __attribute__((ext_vector_type(2)));
                typedef __attribute__((address_space(3))) aq_fp16x4 *lds4;
                const half_t *vp = st + voff + 16 * d + 32 * hh * VD;
                const uint64_t v0 = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)vp));
                const uint64_t v1 = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)(vp + 16 * VD)));
                const half8_t fv = __builtin_bit_cast(half8_t, u64x2_t{v0, v1});
#pragma unroll
                for (int u = 0; u < 2; u++) acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fv, fp[u][hh], acc[u][d], 0, 0, 0);
            }
    };

    if (j_first < j_end) {
        load(j_first), load_mask(j_first + 64 * kg);
        widen(0);
        __syncthreads();
        int stage = 0, j0 = j_first;
        const int kj = 64 * kg; // this wavefront's keys
        auto turn = [&](auto body) __attribute__((always_inline)) {
            const bool more = j0 + AP_KEYS < j_end;
            if (more) load(j0 + AP_KEYS);
            __builtin_amdgcn_sched_barrier(0);
            body();
            __builtin_amdgcn_sched_barrier(0);
            if (more) widen(stage ^ 1);
            __syncthreads();
            stage ^= 1, j0 += AP_KEYS;
        };
        while (j0 + kj + 64 <= w_lean && !coarse) turn([&]() { step(stage, j0 + kj, std::true_type{}); });
        while (j0 + kj < w_end) turn([&]() { step(stage, j0 + kj, std::false_type{}); });
        while (j0 < j_end) turn([]() {}); // blocks that only other wavefronts need
    }
    // ---- the two halves of the keys through LDS: [group of rows][tile of 16][dimensions' tile][lane] four, and references, sums, flags
#pragma unroll
    for (int u = 0; u < 2; u++) {
        l_run[u] = rt_groups_sum(l_run[u]);
        bad[u] |= (uint32_t)__shfl_xor((int)bad[u], 16);
        bad[u] |= (uint32_t)__shfl_xor((int)bad[u], 32);
    }
    float4_t *const rest = (float4_t *)smem;
    float *const sums = (float *)(rest + 8 * NT * 64);
    if (kg == 1) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int d = 0; d < NT; d++) rest[((2 * rg + u) * NT + d) * 64 + lane] = acc[u][d];
            float *const p = sums + (2 * rg + u) * 192 + lane;
            p[0] = m_run[u], p[64] = l_run[u], p[128] = __builtin_bit_cast(float, bad[u]);
        }
    }
    __syncthreads();
    if (kg == 1) return;
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const float *const p = sums + (2 * rg + u) * 192 + lane;
        const float m1 = p[0], top = fmaxf(m_run[u], m1), base = top == -INFINITY ? 0.f : top;
        const float a0 = __builtin_amdgcn_exp2f((m_run[u] - base) * unit), a1 = __builtin_amdgcn_exp2f((m1 - base) * unit), l = l_run[u] * a0 + p[64] * a1;
        const uint32_t bd = bad[u] | __builtin_bit_cast(uint32_t, p[128]);
#pragma unroll
        for (int d = 0; d < NT; d++) {
            const float4_t r = rest[((2 * rg + u) * NT + d) * 64 + lane];
#pragma unroll
            for (int k = 0; k < 4; k++) acc[u][d][k] = fmaf(acc[u][d][k], a0, r[k] * a1);
            if ((bd >> (d >> 1)) & 1u) acc[u][d] = float4_t{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
        }
        const int m = rw + 16 * u + fr;
        if (m >= g.rows) continue;
        if (g.splits > 1) {
            const int64_t at = ((int64_t)bk * g.rows + m) * g.splits + sp;
            if (fg == 0) *(float2_t *)(g.part_ml + 2 * at) = float2_t{top, l};
            if (j_first < j_end) { // (a share with a sum of 0 is not read)
#pragma unroll
                for (int d = 0; d < NT; d++) *(float4_t *)(g.part_o + at * D + 16 * d + 4 * fg) = acc[u][d];
            }
        } else {
            const int qi = m / g.group;
            const float inv = 1.f / l; // no visible key: 0 * inf, NaN
            half_t *const op = g.O + b * g.o_bs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.o_hs + qi * g.o_rs;
#pragma unroll
            for (int d = 0; d < NT; d++) {
                const half4_t o4 = {(half_t)(acc[u][d][0] * inv), (half_t)(acc[u][d][1] * inv), (half_t)(acc[u][d][2] * inv), (half_t)(acc[u][d][3] * inv)};
                *(half4_u *)(op + 16 * d + 4 * fg) = o4;
            }
        }
    }
}

// Joins the shares of a row, four columns a thread: CG threads have the columns of a row, SG groups of them its shares, and the workgroup 256 / (CG SG) rows.  All
// loads are requested at once, and the groups meet in LDS, in a fixed order.  (One thread a column that walked the shares took 20.9 us for 32 rows of 64 shares
// of 128, this 2.9; 4800 rows of 6 shares of 64 with 16 groups, ten of them idle, and a row a workgroup 7.0.)
template <int CG, int SG, bool MASK> __global__ __launch_bounds__(256) void attention_q4_merge_kernel(AttnQ4Args g, int D, int64_t rows) {
    constexpr int R = 256 / (CG * SG), PER = SG < 8 ? 1 : 64 / SG; // (four groups: up to four shares; others 64 at a time)
    __shared__ __attribute__((aligned(16))) float part[R][SG][4 * CG];
    const int t = threadIdx.x, c = t % CG, sg = t / CG % SG, rl = t / (CG * SG);
    const int64_t row = min((int64_t)blockIdx.x * R + rl, rows - 1);
    const bool live = 4 * c < D;
    constexpr float unit = aq_unit(MASK);
    const float *const po = g.part_o + row * g.splits * D + (live ? 4 * c : 0), *const pm = g.part_ml + row * g.splits * 2;
    // this group's shares; one whose sum is 0 has no key, and no outputs were written
    float top = -INFINITY, l = 0.f;
    float4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s0 = 0; s0 < g.splits; s0 += SG * PER) {
        float4_t v[PER];
        float2_t ml[PER];
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (s0 + i * SG < g.splits) { // (uniform)
                const int s = min(s0 + i * SG + sg, g.splits - 1);
                ml[i] = *(const float2_t *)(pm + 2 * s), v[i] = *(const float4_t *)(po + (int64_t)s * D);
            }
        float now = top;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (s0 + i * SG < g.splits) now = fmaxf(now, ml[i][0]);
        const float base = now == -INFINITY ? 0.f : now, old = __builtin_amdgcn_exp2f((top - base) * unit);
        top = now, l *= old;
#pragma unroll
        for (int k = 0; k < 4; k++) y[k] *= old;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (s0 + i * SG < g.splits && s0 + i * SG + sg < g.splits && ml[i][1] != 0.f) {
                const float a = __builtin_amdgcn_exp2f((ml[i][0] - base) * unit);
                l = fmaf(a, ml[i][1], l);
#pragma unroll
                for (int k = 0; k < 4; k++) y[k] = fmaf(a, v[i][k], y[k]);
            }
    }
    __shared__ float mls[R][SG][2];
    *(float4_t *)&part[rl][sg][4 * c] = y;
    if (c == 0) mls[rl][sg][0] = top, mls[rl][sg][1] = l;
    __syncthreads();
    for (int e = t; e < R * D; e += 256) {
        const int rr = e / D, d = e - rr * D;
        const int64_t out = (int64_t)blockIdx.x * R + rr;
        if (out >= rows) break;
        float all = -INFINITY, sum = 0.f, total = 0.f;
#pragma unroll
        for (int s = 0; s < SG; s++) all = fmaxf(all, mls[rr][s][0]);
        const float ref = all == -INFINITY ? 0.f : all;
#pragma unroll
        for (int s = 0; s < SG; s++) {
            const float a = __builtin_amdgcn_exp2f((mls[rr][s][0] - ref) * unit);
            sum = fmaf(part[rr][s][d], a, sum), total = fmaf(mls[rr][s][1], a, total);
        }
        const int bk = (int)(out / g.rows), m = (int)(out - (int64_t)bk * g.rows), b = bk / g.kv_heads, kh = bk - b * g.kv_heads, qi = m / g.group;
        g.O[b * g.o_bs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.o_hs + qi * g.o_rs + d] = (half_t)(sum / total); // no visible key: 0 / 0
    }
}
template <int CG, int SG> static hipError_t launch_aq_merge(const AttnQ4Args &g, int D, int64_t rows, hipStream_t st) {
    constexpr int R = 256 / (CG * SG);
    const dim3 grid((unsigned)((rows + R - 1) / R));
    if (g.mask) hipLaunchKernelGGL((attention_q4_merge_kernel<CG, SG, true>), grid, dim3(256), 0, st, g, D, rows);
    else hipLaunchKernelGGL((attention_q4_merge_kernel<CG, SG, false>), grid, dim3(256), 0, st, g, D, rows);
    return hipGetLastError();
}

// Up to 16 rows per head of keys stream (us, that kernel and the other: 4 x 32 heads on 2001 keys of 96 at 7 rows 15.5 and 24.3, on 2048 of 128 at 8 / 16 rows 22.2 /
// 23.6 and 26.8 / 28.3).
constexpr int AQ_STREAM_ROWS = 16;
static bool aq_streams(int rows) { return rows <= AQ_STREAM_ROWS; }
static int64_t aq_row_tiles(int rows) { return aq_streams(rows) ? 1 : (rows + AP_ROWS - 1) / AP_ROWS; }
// Keys of a workgroup where several share a row tile's, and how many do.
// The streaming kernel: as many as fill the 256 compute units once (a workgroup's eight wavefronts leave no room for a second; two rounds of half the keys, 32 x 8
// heads on 8192 keys of 128: 62 -> 69 us), down to one step each, but two steps (1024 keys) in one launch (32 heads of 80: 8.0 us, in two shares 8.7; four steps 12.3,
// in four shares 9.1; 8 heads on one of 128, 131072 keys: 256 shares 16.4, 64 of four steps 20.1).  More than 128 heads of keys have a share each, so that the last round may leave
// compute units idle (8192 keys of 128: 128 heads 33 us, 136 43, 256 53, 264 89, 512 116): rounds and shares are not weighed against each other here.
// The other: the least of what its rounds of workgroups, the partial results and the second launch take.  A step is some 1.4 + 0.017 head_dim us (2.5, 3.1 and 3.6
// measured at 64, 96 and 128), partial results are written and read at 2.5 TB/s (us for shares: 32 x 128 rows on 1024 keys of 80: 1: 21.3, 4: 16.2, 8: 20.0; 32 x 32 on 544: 1:
// 13.9, 2: 13.6, 5: 10.7; 2 x 4 x 600 on 1373 keys of 64: 3: 21.6, 6: 19.6, 11: 26.4).
static void aq_split(const rt_attention_q4_desc &d, int &splits, int &split_keys) {
    const int rows = d.q_len * (d.heads / d.kv_heads);
    const int64_t stacks = (int64_t)d.batch * d.kv_heads, wgs = stacks * aq_row_tiles(rows);
    const int unit = aq_streams(rows) ? 64 * AQ_WAVES : AP_KEYS, steps = std::max(1, (d.kv_len + unit - 1) / unit);
    int64_t s = 1;
    if (aq_streams(rows)) {
        s = steps <= 2 ? 1 : std::max<int64_t>(1, std::min<int64_t>(steps, 256 / wgs));
    } else if (wgs < 2048) { // (more rounds than eight lose little at their end)
        const double step = 1.4 + 0.017 * d.head_dim, part = (double)stacks * rows * (d.head_dim + 2) * 8 / 2.5e6;
        double best = 0;
        for (int n = 1; n <= std::min(steps, AQ_MAX_SPLITS); n++) {
            const double t = (double)((wgs * n + 255) / 256) * ((steps + n - 1) / n) * step + (n > 1 ? 4 + n * part : 0);
            if (n == 1 || t < best) best = t, s = n;
        }
    }
    const int per = (int)((steps + s - 1) / s);
    splits = (steps + per - 1) / per, split_keys = (int)std::min<int64_t>((int64_t)per * unit, 1 << 30);
}

// A grid's threads along an axis are fewer than 2^32, and the prompt kernel's workgroups, of 512, lie along one.  Shares take no call past that: there are none from 2048
// workgroups on, and at most 64 of a tile (the streaming kernel's lie along the other axis); the join then has at most 2^18 rows.
bool attention_q4_fits(const rt_attention_q4_desc &d) {
    if (d.batch == 0 || d.heads == 0 || d.q_len == 0) return true;
    return aq_row_tiles(d.q_len * (d.heads / d.kv_heads)) * d.batch * d.kv_heads <= 0x7fffff;
}

uint64_t attention_q4_workspace_bytes(const rt_attention_q4_desc &d) {
    if (d.batch == 0 || d.heads == 0 || d.q_len == 0) return 0;
    int splits, keys;
    aq_split(d, splits, keys);
    if (splits <= 1) return 0;
    return (uint64_t)d.batch * d.heads * d.q_len * splits * (d.head_dim + 2) * sizeof(float);
}

template <int NT, int VPR, int MK> static hipError_t launch_aq(const AttnQ4Args &g, dim3 grid, hipStream_t st) {
    using DM = AqDims<NT>;
    constexpr int ROWS = 4 * VPR;
    const size_t wave = (ROWS * 72 + DM::NB * 64) * 2, out = ((size_t)DM::T * VPR * 64 + 2 * ROWS) * sizeof(float);
    const size_t lds = AQ_WAVES * std::max(wave, out);
    if (const hipError_t e = ensure_lds_limit<&attention_q4_kernel<NT, VPR, MK>>(); e != hipSuccess) return e;
    hipLaunchKernelGGL((attention_q4_kernel<NT, VPR, MK>), grid, dim3(64 * AQ_WAVES), lds, st, g);
    return hipGetLastError();
}
template <int NT> static hipError_t launch_aq_rows(const AttnQ4Args &g, dim3 grid, hipStream_t st) {
    if (g.rows <= 4) return g.mask ? launch_aq<NT, 1, 1>(g, grid, st) : launch_aq<NT, 1, 0>(g, grid, st);
    if (g.rows <= 8) return g.mask ? launch_aq<NT, 2, 1>(g, grid, st) : launch_aq<NT, 2, 0>(g, grid, st);
    return g.mask ? launch_aq<NT, 4, 1>(g, grid, st) : launch_aq<NT, 4, 0>(g, grid, st);
}
template <int NT, int MK> static hipError_t launch_aq_tile(const AttnQ4Args &g, unsigned wgs, hipStream_t st) {
    constexpr size_t ring = (size_t)2 * aq_stage(NT) * sizeof(half_t) + 16 * sizeof(uint32_t), halves = (size_t)8 * (NT * 64 * 16 + 192 * 4), lds = ring > halves ? ring : halves;
    if (const hipError_t e = ensure_lds_limit<&attention_q4_tile_kernel<NT, MK>>(); e != hipSuccess) return e;
    hipLaunchKernelGGL((attention_q4_tile_kernel<NT, MK>), dim3(wgs), dim3(512), lds, st, g);
    return hipGetLastError();
}

hipError_t launch_attention_q4(const rt_attention_q4_desc &d, const void *q, const void *k_cache, const void *v_cache, const void *mask,
                               const int32_t *kv_lens, void *out, void *workspace, uint64_t workspace_bytes, hipStream_t stream, const DeviceInfo &dev) {
    AttnQ4Args g{};
    const uint64_t soff = cache_q4_scale_offset(d.batch, d.kv_heads, d.capacity, d.head_dim);
    g.Q = (const half_t *)q, g.O = (half_t *)out, g.mask = mask, g.lens = kv_lens;
    g.Kc = (const uint8_t *)k_cache, g.Vc = (const uint8_t *)v_cache;
    g.Ks = (const half_t *)(g.Kc + soff), g.Vs = (const half_t *)(g.Vc + soff);
    g.q_bs = d.q_strides[0], g.q_hs = d.q_strides[1], g.q_rs = d.q_strides[2];
    g.o_bs = d.o_strides[0], g.o_hs = d.o_strides[1], g.o_rs = d.o_strides[2];
    g.m_bs = d.mask_strides[0], g.m_rs = d.mask_strides[1], g.mask_f32 = d.mask_dtype == RT_F32;
    g.kv_heads = d.kv_heads, g.group = d.heads / d.kv_heads, g.rows = d.q_len * g.group;
    g.kv_len = d.kv_len, g.q_len = d.q_len, g.capacity = d.capacity, g.causal = d.causal;
    g.scale = d.scale, g.scale_log2e = d.scale * kLog2eQ4;
    aq_split(d, g.splits, g.split_keys);
    const uint64_t need = attention_q4_workspace_bytes(d);
    if (need && workspace && workspace_bytes >= need && !((uintptr_t)workspace & 15u)) {
        g.part_o = (float *)workspace, g.part_ml = g.part_o + (uint64_t)d.batch * d.heads * d.q_len * g.splits * d.head_dim;
    } else {
        g.splits = 1, g.split_keys = std::max(d.kv_len, 1);
    }
    const int64_t tiles = aq_row_tiles(g.rows), stacks = (int64_t)d.batch * d.kv_heads;
    g.row_tiles = (int)tiles;
    const dim3 grid((unsigned)g.splits, (unsigned)stacks);
    auto go = [&](auto nt) -> hipError_t {
        constexpr int NT = decltype(nt)::value;
        if (aq_streams(g.rows)) return launch_aq_rows<NT>(g, grid, stream);
        const unsigned wgs = (unsigned)(tiles * stacks * g.splits);
        return !mask ? launch_aq_tile<NT, 0>(g, wgs, stream) : g.mask_f32 ? launch_aq_tile<NT, 1>(g, wgs, stream) : launch_aq_tile<NT, 2>(g, wgs, stream);
    };
    hipError_t e;
    switch (d.head_dim / 16) {
    case 1: e = go(std::integral_constant<int, 1>{}); break;
    case 2: e = go(std::integral_constant<int, 2>{}); break;
    case 3: e = go(std::integral_constant<int, 3>{}); break;
    case 4: e = go(std::integral_constant<int, 4>{}); break;
    case 5: e = go(std::integral_constant<int, 5>{}); break;
    case 6: e = go(std::integral_constant<int, 6>{}); break;
    case 7: e = go(std::integral_constant<int, 7>{}); break;
    default: e = go(std::integral_constant<int, 8>{}); break;
    }
    if (e != hipSuccess || g.splits <= 1) return e;
    const int64_t rows = stacks * g.rows;
    if (d.head_dim <= 64) return g.splits <= 4 ? launch_aq_merge<16, 4>(g, d.head_dim, rows, stream) : g.splits <= 8 ? launch_aq_merge<16, 8>(g, d.head_dim, rows, stream) : launch_aq_merge<16, 16>(g, d.head_dim, rows, stream);
    return g.splits <= 4 ? launch_aq_merge<32, 4>(g, d.head_dim, rows, stream) : launch_aq_merge<32, 8>(g, d.head_dim, rows, stream);
}

} // namespace rt
