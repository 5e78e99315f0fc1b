// Attention of sequences of different lengths, many query rows: prompts that lie packed one behind another, and rows against a cache held in pages (ragged.h).
//
//   out[r, h] = sum_j p_j v_j,  p = softmax_j(scale * q[r, h] . k_j) over the keys j that row r sees
//
// The rows of the heads that share a head of keys are one matrix, row m = query row * group + head of the group, so that a block of keys and values is read
// once for all of them.  A workgroup has 128 such rows of a sequence, a wavefront 32, against blocks of 64 keys that go from memory straight into LDS (no registers; two stages of the
// ring at head_dim above 64, three below), rows of 64 or 128 halves, 16-byte chunks XOR-swizzled by the row.  Four wavefronts and two workgroups on a compute unit where there are
// enough of them, else eight wavefronts, of which four have the other 64 of 128 keys, and the halves meet at the end (rr_plan).
//   S^T = K Q^T, v_mfma_f32_32x32x16_f16 with the keys as first operand: a lane has 16 of a tile's 32 keys of one row, and its neighbour 32 lanes on the others.
//   softmax: scores stay as the product has them; p = exp2(s * sc - c) with the row's running reference c (RG_BELOW).  Sums and references are f32; probabilities enter the
//     second product as f16 and the sum is that of the rounded ones.
//   O^T += V^T P^T: eight probabilities of a lane are an operand as they lie, in an order of keys of their own; the values' operand comes in that order, transposed, out of
//     LDS (ds_read_b64_tr_b16).
// Which tile of which sequence a workgroup has it finds out by itself (rg_locate): the host knows no lengths.
//
// Prompts of 4096 to 1792 rows, 32 heads on 8 of 128, causal, 308 GFLOP: 365 us, 843 TFLOP/s, at 1.9 GHz, which is what the package's power leaves (the library's product of 8192^3 1140).  Matrix
// instructions run 41 % of the cycles, vector ones 36 %; the rest are waits for LDS and of two wavefronts for one unit.  Without its loads the kernel takes 16 % less, which is
// not their latency (with half a step more for the values, and a second barrier, it took 2 % more), without its exponentials 4 %.
// Scores of the next block beside this block's probabilities, so that both units work for one wavefront, need 64 registers more, and with them in scratch or remade took 6 to 20 % longer.
#include "ragged.h"

#include <algorithm>
#include <cmath>

namespace rt {

constexpr int RR_ROWS = 128, RR_KEYS = 64; // rows of a workgroup; keys of a wavefront's block
constexpr int RR_MAX_SPLITS = 64;
constexpr int rr_pitch(int ks) { return ks <= 4 ? 64 : 128; } // halves of a row in LDS
constexpr int rr_stages(int ks) { return ks <= 4 ? 3 : 2; } // (with three of 16 KB, and registers for three wavefronts of a SIMD, three workgroups share a compute unit: prompts of up to 4096 rows, 32 heads on 8 of 64, 235 -> 216 us)
typedef __fp16 rr_fp16x4 __attribute__((ext_vector_type(4)));
typedef half_t half4_ru __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ constexpr int rr_waitcnt(int n) { return 0x0070 | (n & 0xF) | (((n >> 4) & 0x3) << 14); } // vmcnt(n) lgkmcnt(0)

// What chunk numbers of row r are XORed with.  The reads of keys take one chunk of 32 rows, those of values 64 bytes of four neighbouring rows (and of four others): rows four apart differ
// in the low bits and neighbours in the high ones, so that each covers the banks evenly.
template <int PITCH> __device__ __forceinline__ int rr_swizzle(int r) {
    return PITCH == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// maximum / sum of lanes l and l ^ 32
__device__ __forceinline__ float rr_pair_max(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
}
__device__ __forceinline__ float rr_pair_sum(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)a[0]) + __builtin_bit_cast(float, (uint32_t)a[1]);
}

// KS: steps of 16 over head_dim (the last one may be half).  NH: groups of four wavefronts, each with its 64 keys of a step
template <int KS, bool PAGED, int NH> __global__ __launch_bounds__(256 * NH, KS <= 4 && NH == 1 ? 3 : 2) void attention_ragged_kernel(RaggedArgs g) {
    constexpr int RR_STEP = RR_KEYS * NH, WAVES = 4 * NH;
    constexpr int P = rr_pitch(KS), CPR = P / 8, DT = (KS + 1) / 2, STAGES = rr_stages(KS);
    constexpr int BLK = RR_STEP * P;              // halves of a step's keys (or values)
    constexpr int RPI = 64 / CPR;                 // rows of a load instruction
    constexpr int NI = RR_STEP / RPI / WAVES;         // of them a wavefront issues per step and tensor
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const half_t *const ring = (const half_t *)smem; // [STAGES][keys | values][RR_STEP][P]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int r = lane & 31, hi = lane >> 5, rg = wave & 3, half = wave >> 2; // group of rows, of wavefronts

    int b, tile, first, n, key0;
    const int line = blockIdx.x / g.kv_heads, kh = blockIdx.x - line * g.kv_heads, place = line / g.splits, share = line - place * g.splits;
    if (!rg_locate<RR_ROWS>(g, place, b, tile, first, n)) return;
    b = __builtin_amdgcn_readfirstlane(b), tile = __builtin_amdgcn_readfirstlane(tile), n = __builtin_amdgcn_readfirstlane(n);
    int all_keys;
    const int len = __builtin_amdgcn_readfirstlane(rg_keys<PAGED>(g, b, key0, all_keys));
    first = __builtin_amdgcn_readfirstlane(first), key0 = __builtin_amdgcn_readfirstlane(key0);
    const int rows = n * g.group, off = __builtin_amdgcn_readfirstlane(all_keys - rg_all_rows(g, b, first)); // causal: query row i sees keys up to i + off
    const int row0 = tile * RR_ROWS, rw = row0 + 32 * rg;
    const int q0 = row0 / g.group, over = row0 - q0 * g.group; // (the tile's other query rows are found from its first without a division)
    auto query = [&](int m) { return q0 + rg_query(g, m - row0 + over); };
    auto sees = [&](int m) { return g.causal ? max(0, min(len, query(min(m, rows - 1)) + off + 1)) : len; }; // keys that row m sees: the first so many
    // this share's steps of those that a row of the tile sees
    const int nkb = (sees(row0 + RR_ROWS - 1) + RR_STEP - 1) / RR_STEP;
    const int kb0 = __builtin_amdgcn_readfirstlane((int)((int64_t)nkb * share / g.splits)), kb1 = __builtin_amdgcn_readfirstlane((int)((int64_t)nkb * (share + 1) / g.splits));
    const int seen_all = __builtin_amdgcn_readfirstlane(rw < rows ? sees(rw) : 0), seen_any = __builtin_amdgcn_readfirstlane(rw < rows ? sees(rw + 31) : 0); // by each, by any of the wavefront's rows

    // queries: row rw + r, dimensions 16 k + 8 hi .. + 7
    const int m = min(rw + r, rows - 1), qi = query(m), qh = kh * g.group + (m - qi * g.group);
    const int last = min(len - 1, g.causal ? qi + off : len - 1);
    half8_t fq[KS];
    auto queries = [&]() __attribute__((always_inline)) {
        const half_t *q = g.Q + (int64_t)(first + qi) * g.q_rs + (int64_t)qh * g.q_hs;
        const half_t sign = (half_t)g.sign;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int d = 16 * k + 8 * hi;
            fq[k] = d < g.D ? *(const half8_t *)(q + d) * half8_t{sign, sign, sign, sign, sign, sign, sign, sign} : half8_t{};
        }
        // awaited here: a first use in the loop would wait there, for these and with them for every load into LDS
#pragma unroll
        for (int k = 0; k < KS; k++) asm volatile("" : "+v"(fq[k]));
    };

    // Of the columns behind head_dim, which no load writes, the products read those up to the next 32: they are zeros
    if (g.D < 32 * DT) {
        for (int i = t; i < STAGES * 2 * BLK / 8; i += 64 * WAVES) ((uint4_t *)smem)[i] = uint4_t{0, 0, 0, 0};
        __syncthreads();
    }

    // ---- loads: instruction i of this wavefront brings the rows RPI (wave + WAVES i) .. of the step's; lane l the chunk l % CPR of row l / CPR.  All of its instructions are at the same
    // row of 16, so that offsets, chunks and lanes are the same for all, and only the 16 rows' address differs
    const int row16 = (RPI * wave) & 15, lrow = row16 + lane / CPR, c = 8 * ((lane % CPR) ^ rr_swizzle<P>(lrow));
    const uint64_t lanes = __builtin_amdgcn_ballot_w64(c < g.D); // whose chunk is a part of the row
    const half_t *const K = g.K + (int64_t)kh * g.k_hs, *const V = g.V + (int64_t)kh * g.v_hs;
    typedef __attribute__((address_space(4))) const int32_t *scalar_t; // read through the scalar cache: no vector load is awaited for them
    const scalar_t table = PAGED ? (scalar_t)(uintptr_t)(g.table + b * g.table_stride) : (scalar_t)0;
    const int last_entry = PAGED ? max(0, len - 1) >> g.page_shift : 0;
    int pages[NI], own[4]; // of the 16 rows each that this wavefront brings, and of those that it multiplies
    auto look = [&](int kb) __attribute__((always_inline)) {
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < NI; i++) pages[i] = table[min((kb * RR_STEP + RPI * (wave + WAVES * i)) >> g.page_shift, last_entry)];
#pragma unroll
            for (int i = 0; i < 4; i++) own[i] = table[min((kb * RR_STEP + RR_KEYS * half + 16 * i) >> g.page_shift, last_entry)];
        }
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)smem;
    const uint32_t k_off = 2u * ((uint32_t)lrow * (uint32_t)(PAGED ? g.D : g.k_rs) + (uint32_t)c), v_off = 2u * ((uint32_t)lrow * (uint32_t)(PAGED ? g.D : g.v_rs) + (uint32_t)c);
    // step kb into a stage, from the pages that `pages` has; -> whether this wavefront's four times 16 keys are there, as bits
    auto issue = [&](int stage, int kb) __attribute__((always_inline)) {
        uint32_t there = 15u;
        const int j0 = kb * RR_STEP;
        const bool part = !PAGED && j0 + RR_STEP > len; // of rows behind the last of packed keys the last is read again
        const half_t *const k0 = K + (int64_t)(key0 + j0) * g.k_rs, *const v0 = V + (int64_t)(key0 + j0) * g.v_rs;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int row = RPI * (wave + WAVES * i) - row16; // of the step: a multiple of 16
            const half_t *kp, *vp;
            uint32_t ko = k_off, vo = v_off;
            if constexpr (PAGED) {
                const int page = (uint32_t)pages[i] < (uint32_t)g.pages ? pages[i] : 0;
                const int64_t at = (int64_t)page * g.k_rs + (int64_t)(((j0 + row) & ((1 << g.page_shift) - 1)) * g.D);
                kp = K + at, vp = V + at;
            } else if (part) {
                const uint32_t j = (uint32_t)min(row + lrow, len - 1 - j0);
                kp = k0, vp = v0;
                ko = 2u * (j * (uint32_t)g.k_rs + (uint32_t)c), vo = 2u * (j * (uint32_t)g.v_rs + (uint32_t)c);
            } else {
                kp = k0 + row * g.k_rs, vp = v0 + row * g.v_rs;
            }
            const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)(2 * (stage * 2 * BLK + (row + row16) * P)));
            // (every lane is active here, and is again)
            asm volatile("s_mov_b64 exec, %6\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\t"
                         "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %5\n\ts_mov_b64 exec, -1" ::"s"(dst),
                         "s"(dst + 2 * BLK), "v"(ko), "s"(kp), "v"(vo), "s"(vp), "s"(lanes)
                         : "m0", "memory");
        }
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if ((uint32_t)own[i] >= (uint32_t)g.pages) there &= ~(1u << i);
        }
        return there;
    };
    // all but the newest `keep` blocks' loads of this wavefront have landed, and its LDS reads have returned; then everybody's have
    auto publish = [&](auto keep) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(rr_waitcnt(decltype(keep)::value * 2 * NI));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    float16_t acc[DT];
    float c_run = -INFINITY, l_run = 0.f; // the reference, this lane's share of the sum
    bool coarse = false; // whether scores are rounded before the reference is taken away (uniform)
#pragma unroll
    for (int d = 0; d < DT; d++) acc[d] = float16_t{};

    // fragment offsets in a stage, halves
    int koff[KS], voff[DT][2];
#pragma unroll
    for (int k = 0; k < KS; k++) koff[k] = r * P + 8 * ((2 * k + hi) ^ rr_swizzle<P>(r));
    auto value_at = [&](int d, int w) { // dimensions 32 d .., of 16 keys the row 4 hi + (lane % 16) / 4, and 8 more
        const int s = lane & 15, half = (lane >> 4) & 1, row = 4 * hi + (s >> 2) + 8 * w;
        return BLK + row * P + 8 * ((4 * d + 2 * half + ((s & 3) >> 1)) ^ rr_swizzle<P>(row)) + 4 * (s & 1);
    };
#pragma unroll
    for (int d = 0; d < DT; d++) voff[d][0] = value_at(d, 0), voff[d][1] = value_at(d, 1);
    auto transposed = [&](const half_t *p0, const half_t *p1) __attribute__((always_inline)) {
        typedef uint64_t u64x2_t __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) rr_fp16x4 *lds4;
        const uint64_t v0 = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)p0));
        const uint64_t v1 = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)p1));
        return __builtin_bit_cast(half8_t, u64x2_t{v0, v1});
    };
    auto values = [&](const half_t *st, int d, int s) __attribute__((always_inline)) { // dimensions 32 d .., keys 16 s ..
        return transposed(st + voff[d][0] + 16 * s * P, st + voff[d][1] + 16 * s * P);
    };

    auto step = [&](int stage, int kb, uint32_t there, auto lean_c) __attribute__((always_inline)) {
        constexpr bool LEAN = decltype(lean_c)::value;
        const half_t *const st = ring + stage * 2 * BLK + half * RR_KEYS * P;
        const int j0 = kb * RR_STEP + half * RR_KEYS; // this wavefront's first key
        // Operands are read four ahead of the products that take them: left to itself the compiler reads each right before its product, and waits
        float16_t S[2] = {};
        half8_t ahead[2][4];
        auto keys = [&](int i) __attribute__((always_inline)) { return *(const half8_t *)(st + koff[(i / 2) % KS] + 32 * (i & 1) * P); }; // of products 0 .. 2 KS - 1: both tiles of 32 keys in turn
#pragma unroll
        for (int i = 0; i < 4 && i < 2 * KS; i++) ahead[0][i] = keys(i);
#pragma unroll
        for (int q = 0; q < (2 * KS + 3) / 4; q++) {
#pragma unroll
            for (int i = 4 * q + 4; i < 4 * q + 8 && i < 2 * KS; i++) ahead[(q + 1) & 1][i & 3] = keys(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 4 * q; i < 4 * q + 4 && i < 2 * KS; i++) S[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[q & 1][i & 3], fq[i / 2], S[i & 1], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        half8_t next[2][DT];
        if constexpr (LEAN)
#pragma unroll
            for (int d = 0; d < DT; d++) next[0][d] = values(st, d, 0);
        __builtin_amdgcn_sched_barrier(0);
        // register i of S[u]: key 32 u + 8 (i / 4) + 4 hi + i % 4 of the block
        int left = last - j0 - 4 * hi;
        auto sees_key = [&](int u, int i) { return 32 * u + 8 * (i >> 2) + (i & 3) <= left && ((there >> (2 * u + (i >> 3))) & 1u); };
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if constexpr (!LEAN) S[u][i] = sees_key(u, i) ? S[u][i] : -INFINITY;
                top = fmaxf(top, S[u][i]);
            }
        top = rr_pair_max(top) * g.sc;
        float sc = g.sc;
        if (__builtin_amdgcn_ballot_w64(top - c_run > RG_ABOVE)) {
            const float c = fmaxf(c_run, top - RG_BELOW), alpha = c == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(c_run - c);
            c_run = c;
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] *= alpha;
            // The reference is a rounded product, which a score meets in the fused multiply-add without a rounding of its own: past 4096 the difference shows, and past 2^24 a
            // probability could leave f16.  From there on scores are rounded first.
            coarse = __builtin_amdgcn_ballot_w64(c != -INFINITY && !(__builtin_fabsf(c) < 4096.f)) != 0;
        }
        if (coarse) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 16; i++) S[u][i] *= sc;
            sc = 1.f;
        }
        const float c = c_run == -INFINITY ? 0.f : c_run; // a row that has seen no key: exp2(-inf)
        half8_t fp[4];
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const half2_t p = {(half_t)__builtin_amdgcn_exp2f(fmaf(S[u][i], sc, -c)), (half_t)__builtin_amdgcn_exp2f(fmaf(S[u][i + 1], sc, -c))};
                sum = __builtin_amdgcn_fdot2(p, half2_t{(half_t)1, (half_t)1}, sum, false);
                fp[2 * u + (i >> 3)][i & 7] = p[0], fp[2 * u + (i >> 3)][(i & 7) + 1] = p[1];
            }
        l_run += sum;
        bool odd = false;
        if constexpr (!LEAN) { // a value that is not finite must not reach, as 0 * inf, the rows that do not see its key
            float x = 0.f;
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    x = rg_odd(values(st, d, s), x);
                    __builtin_amdgcn_sched_barrier(0);
                }
            odd = __builtin_amdgcn_ballot_w64(x != 0.f) != 0; // (NaN is)
        }
        if (!LEAN && odd) {
            // Such values enter as 0, and a second product counts, for each row and dimension, how many it sees that are +inf (1 each), -inf (256) or NaN (both)
#pragma unroll
            for (int d = 0; d < DT; d++) {
                float16_t mark = {};
                asm volatile("" : "+v"(left), "+s"(there)::"memory"); // (read and compared again: nothing of this is worth registers outside)
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    half8_t v = values(st, d, s), vis;
                    const half8_t code = rg_take_odd(v);
#pragma unroll
                    for (int e = 0; e < 8; e++) vis[e] = __builtin_bit_cast(half_t, (uint16_t)(sees_key(s >> 1, 8 * (s & 1) + e) ? 0x3C00 : 0));
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, fp[s], acc[d], 0, 0, 0);
                    mark = __builtin_amdgcn_mfma_f32_32x32x16_f16(code, vis, mark, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    acc[d][i] += (int)mark[i] & 255 ? INFINITY : 0.f;
                    acc[d][i] += mark[i] >= 256.f ? -INFINITY : 0.f;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            if constexpr (!LEAN)
#pragma unroll
                for (int d = 0; d < DT; d++) next[0][d] = values(st, d, 0);
#pragma unroll
            for (int s = 0; s < 4; s++) {
                if (s < 3)
#pragma unroll
                    for (int d = 0; d < DT; d++) next[(s + 1) & 1][d] = values(st, d, s + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < DT; d++) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(next[s & 1][d], fp[s], acc[d], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };

    if (kb0 < kb1) {
        uint32_t there[STAGES];
        look(kb0);
#pragma unroll
        for (int s = 0; s < STAGES - 1; s++) {
            there[s] = issue(s, min(kb0 + s, kb1 - 1)); // past the end: the last block again, into a stage that nobody reads
            look(min(kb0 + s + 1, kb1 - 1));
        }
        queries(); // behind the first blocks' loads: the trips to memory are one
        publish(std::integral_constant<int, STAGES - 2>{});
        int cur = 0, fill = STAGES - 1, kb = kb0;
        auto turn = [&](auto body) __attribute__((always_inline)) {
            const uint32_t now = there[0];
#pragma unroll
            for (int s = 0; s + 2 < STAGES; s++) there[s] = there[s + 1];
            there[STAGES - 2] = issue(fill, min(kb + STAGES - 1, kb1 - 1));
            look(min(kb + STAGES, kb1 - 1));
            body(now);
            publish(std::integral_constant<int, STAGES - 2>{});
            cur = cur + 1 == STAGES ? 0 : cur + 1, fill = fill + 1 == STAGES ? 0 : fill + 1;
            kb++;
        };
        // steps of which each of the wavefront's rows sees all of its keys, of which any sees one
        const int lean = min(kb1, (seen_all / RR_KEYS + NH - 1 - half) / NH), any = min(kb1, ((seen_any + RR_KEYS - 1) / RR_KEYS + NH - 1 - half) / NH);
        while (kb < lean && there[0] == 15u) turn([&](uint32_t) { step(cur, kb, 15u, std::true_type{}); });
        while (kb < any) turn([&](uint32_t now) { step(cur, kb, now, std::false_type{}); });
        while (kb < kb1) turn([](uint32_t) {}); // blocks that only other wavefronts need
    }
    __builtin_amdgcn_s_waitcnt(rr_waitcnt(0)); // nothing lands after the workgroup has ended
    float l = rr_pair_sum(l_run);
    if constexpr (NH == 2) { // the two halves of the keys through LDS: [group of rows][reference, sum, outputs][lane]
        __syncthreads();
        float *const other = (float *)smem + rg * (2 + 16 * DT) * 64 + lane;
        if (half) {
            other[0] = c_run, other[64] = l;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) other[(2 + 16 * d + i) * 64] = acc[d][i];
        }
        __syncthreads();
        if (half) return;
        const float c1 = other[0], top = fmaxf(c_run, c1), base = top == -INFINITY ? 0.f : top;
        const float a0 = __builtin_amdgcn_exp2f(c_run - base), a1 = __builtin_amdgcn_exp2f(c1 - base);
        l = l * a0 + other[64] * a1, c_run = top;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[d][i] = fmaf(acc[d][i], a0, other[(2 + 16 * d + i) * 64] * a1);
    }
    if (rw + r >= rows) return;
    const int64_t row = first + qi;
    if (g.splits > 1) {
        const int64_t at = ((row * g.kv_heads + kh) * g.group + (m - qi * g.group)) * g.splits + share;
        if (hi == 0) *(float2_t *)(g.part_ml + 2 * at) = float2_t{c_run, l};
        if (kb0 < kb1) { // (a share with a sum of 0 is not read)
            float *const po = g.part_o + at * g.D;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int x = 32 * d + 2 * i + 4 * hi;
                    if (x < g.D) *(float4_t *)(po + x) = float4_t{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
                }
        }
    } else {
        const float inv = 1.f / l; // no visible key: 0 * inf, NaN
        half_t *const o = g.O + row * g.o_rs + (int64_t)qh * g.o_hs;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int x = 32 * d + 2 * i + 4 * hi;
                if (x < g.D) *(half4_ru *)(o + x) = half4_ru{(half_t)(acc[d][i] * inv), (half_t)(acc[d][i + 1] * inv), (half_t)(acc[d][i + 2] * inv), (half_t)(acc[d][i + 3] * inv)};
            }
    }
}

// Joins the shares of a row in a fixed order: 32 lanes a row, which have a share's weight each (two past 32 shares) and then four columns, eight shares' loads at a time.  A workgroup has
// RJ_ROWS of a tile's rows (blockIdx.y).
constexpr int RJ_ROWS = 8;
__global__ __launch_bounds__(32 * RJ_ROWS) void attention_ragged_join_kernel(RaggedArgs g) {
    int b, tile, first, n;
    const int place = blockIdx.x / g.kv_heads, kh = blockIdx.x - place * g.kv_heads;
    if (!rg_locate<RR_ROWS>(g, place, b, tile, first, n)) return;
    const int rows = n * g.group, m0 = tile * RR_ROWS + blockIdx.y * RJ_ROWS;
    if (m0 >= rows) return;
    const int c = threadIdx.x & 31, m = min(m0 + (int)(threadIdx.x >> 5), rows - 1); // (all lanes stay: they exchange)
    const int qi = m / g.group, h = kh * g.group + (m - qi * g.group);
    const int64_t row = first + qi, at = (row * g.kv_heads * g.group + h) * g.splits;
    float2_t ml[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        ml[i] = *(const float2_t *)(g.part_ml + 2 * (at + min(c + 32 * i, g.splits - 1)));
        if (c + 32 * i >= g.splits) ml[i] = float2_t{-INFINITY, 0.f};
    }
    float top = fmaxf(ml[0][0], ml[1][0]);
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float base = top == -INFINITY ? 0.f : top;
    float w[2], l;
#pragma unroll
    for (int i = 0; i < 2; i++) w[i] = __builtin_amdgcn_exp2f(ml[i][0] - base);
    l = w[0] * ml[0][1] + w[1] * ml[1][1];
#pragma unroll
    for (int x = 16; x; x >>= 1) l += __shfl_xor(l, x);
    const float *const po = g.part_o + at * g.D + (4 * c < g.D ? 4 * c : 0);
    float4_t y = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < g.splits; s0 += 8) {
        float4_t v[8];
        float a[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int s = min(s0 + i, g.splits - 1), from = (threadIdx.x & 32) + (s & 31);
            v[i] = *(const float4_t *)(po + (int64_t)s * g.D);
            const float sum = s < 32 ? __shfl(ml[0][1], from) : __shfl(ml[1][1], from); // (s is the same in all lanes)
            a[i] = s < 32 ? __shfl(w[0], from) : __shfl(w[1], from);
            if (s0 + i >= g.splits || sum == 0.f) a[i] = 0.f, v[i] = float4_t{0.f, 0.f, 0.f, 0.f}; // (no key: no outputs were written)
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = fmaf(a[i], v[i][k], y[k]);
    }
    if (m0 + (int)(threadIdx.x >> 5) >= rows || 4 * c >= g.D) return;
    const float inv = 1.f / l; // no visible key: 0 * inf, NaN
    *(half4_ru *)(g.O + row * g.o_rs + (int64_t)h * g.o_hs + 4 * c) = half4_ru{(half_t)(y[0] * inv), (half_t)(y[1] * inv), (half_t)(y[2] * inv), (half_t)(y[3] * inv)};
}

// Tiles of a call, at most: sequences have `rows` rows in all, and each may leave one tile begun.
static int64_t rr_tiles(int batch, int group, int rows, int max_rows) {
    return std::min<int64_t>((int64_t)batch * (((int64_t)max_rows * group + RR_ROWS - 1) / RR_ROWS), (int64_t)rows * group / RR_ROWS + batch);
}
// Groups of wavefronts of a workgroup, and shares of a row's keys.
struct RaggedPlan {
    int groups, splits;
};
// From 512 workgroups on two of four wavefronts fill each compute unit; where the causal flag makes tiles of unlike lengths the longest of fewer of them end last, alone, and eight wavefronts
// on each are faster (us, four and eight: 2048 rows of 24 heads of 96, 384 tiles, 48.8 and 41.7; without the flag, 4 x 1500 rows of six heads of 64, 288 tiles, 36.7 and 43.8), as
// they are where there is no second workgroup (512 rows on 4096 keys, 32 heads on 8 of 128, 208 tiles, 88.4 and 81.5).  Short ones do not pay for the join of the halves (24 prompts of up to
// 100 rows 8.6 and 9.6).
// (256 compute units are the card's; the workspace is asked for without a device to look at.)
// Shares: the least of what the steps, the partial results and the second launch take.  A step of 128 keys is some 0.5 + 0.016 head_dim us, partial results are written and read at 2.5 TB/s.  Tiles of one
// length take rounds of workgroups; with the causal flag they are of unlike lengths, and take what the longest takes, or all of them on 256 compute units (5088 rows of four heads on one of
// 96, 160 tiles: 70 us in one share, 58 in three).
static RaggedPlan rr_plan(int64_t wgs, int heads, int rows, int max_rows, int max_keys, int head_dim, int causal) {
    RaggedPlan p{1, 1};
    const int64_t steps = (max_keys + 2 * RR_KEYS - 1) / (2 * RR_KEYS);
    if (steps > 2 && (wgs <= 256 || (causal && wgs < 512))) p.groups = 2;
    if (p.groups == 2 && wgs <= 256) {
        const double step = 0.5 + 0.016 * head_dim, part = (double)rows * heads * (head_dim + 2) * 8 / 2.5e6;
        double best = 0;
        for (int n = 1; n <= std::min<int64_t>(steps, RR_MAX_SPLITS); n++) {
            const double per = (double)((steps + n - 1) / n), all = (double)wgs * steps / 256 * (1 - 0.5 * std::min(max_rows, max_keys) / max_keys);
            const double t = (causal ? std::max(per, all) : (double)((wgs * n + 255) / 256) * per) * step + (n > 1 ? 6 + n * part : 0);
            if (n == 1 || t < best) best = t, p.splits = n;
        }
    }
    return p;
}
static uint64_t rr_workspace(int heads, int rows, int head_dim, int splits) {
    return splits <= 1 ? 0 : (uint64_t)rows * heads * splits * (head_dim + 2) * sizeof(float);
}

bool ragged_fits(int batch, int kv_heads, int group, int rows, int max_rows) {
    return rr_tiles(batch, group, rows, max_rows) * kv_heads <= 0x7fffff; // a grid's threads are fewer than 2^32; shares take no call past that
}
uint64_t ragged_workspace_bytes(int batch, int heads, int kv_heads, int rows, int max_rows, int max_keys, int head_dim, int causal) {
    return rr_workspace(heads, rows, head_dim, rr_plan(rr_tiles(batch, heads / kv_heads, rows, max_rows) * kv_heads, heads, rows, max_rows, max_keys, head_dim, causal).splits);
}

template <int KS, bool PAGED, int NH> static hipError_t launch_rr(const RaggedArgs &g, hipStream_t st) {
    constexpr size_t lds = (size_t)rr_stages(KS) * 2 * NH * RR_KEYS * rr_pitch(KS) * sizeof(half_t);
    if (const hipError_t e = ensure_lds_limit<&attention_ragged_kernel<KS, PAGED, NH>>(); e != hipSuccess) return e;
    hipLaunchKernelGGL((attention_ragged_kernel<KS, PAGED, NH>), dim3((unsigned)((int64_t)g.tiles * g.kv_heads * g.splits)), dim3(256 * NH), lds, st, g);
    return hipGetLastError();
}

// exp(scale * s) as exp2(sc * s) with sc above 0, whatever the scale's sign; a scale of 0 leaves scores of 0
void ragged_scale(RaggedArgs &g, float scale) {
    g.sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
    g.sc = scale == 0.f ? 1.f : std::fabs(scale) * kLog2eR;
    g.per_group = 1.f / g.group;
}

// `g` has the operands; the shares, and where partial results go, are chosen here.
hipError_t launch_ragged(RaggedArgs &g, bool paged, void *workspace, uint64_t workspace_bytes, hipStream_t stream) {
    g.tiles = (int)rr_tiles(g.batch, g.group, g.rows, g.max_rows);
    const RaggedPlan plan = rr_plan((int64_t)g.tiles * g.kv_heads, g.kv_heads * g.group, g.rows, g.max_rows, g.max_keys, g.D, g.causal);
    g.splits = plan.splits;
    const uint64_t need = rr_workspace(g.kv_heads * g.group, g.rows, g.D, g.splits);
    if (need && workspace && workspace_bytes >= need && !((uintptr_t)workspace & 15u))
        g.part_o = (float *)workspace, g.part_ml = g.part_o + (uint64_t)g.rows * g.kv_heads * g.group * g.splits * g.D;
    else
        g.splits = 1;
    auto go = [&](auto ks) -> hipError_t {
        constexpr int KS = decltype(ks)::value;
        if (plan.groups == 2) return paged ? launch_rr<KS, true, 2>(g, stream) : launch_rr<KS, false, 2>(g, stream);
        return paged ? launch_rr<KS, true, 1>(g, stream) : launch_rr<KS, false, 1>(g, stream);
    };
    hipError_t e;
    switch ((g.D + 15) / 16) {
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
    hipLaunchKernelGGL(attention_ragged_join_kernel, dim3((unsigned)((int64_t)g.tiles * g.kv_heads), RR_ROWS / RJ_ROWS), dim3(32 * RJ_ROWS), 0, stream, g);
    return hipGetLastError();
}

bool attention_packed_fits(const rt_attention_packed_desc &d) {
    if (d.batch == 0 || d.heads == 0 || d.rows == 0) return true;
    return ragged_fits(d.batch, d.kv_heads, d.heads / d.kv_heads, d.rows, d.max_rows);
}
uint64_t attention_packed_workspace_bytes(const rt_attention_packed_desc &d) {
    if (d.batch == 0 || d.heads == 0 || d.rows == 0) return 0;
    return ragged_workspace_bytes(d.batch, d.heads, d.kv_heads, d.rows, d.max_rows, d.max_keys, d.head_dim, d.causal);
}
hipError_t launch_attention_packed(const rt_attention_packed_desc &d, const void *q, const void *k, const void *v, const int32_t *starts, const int32_t *kv_starts,
                                   void *out, void *workspace, uint64_t workspace_bytes, hipStream_t stream) {
    RaggedArgs g{};
    g.Q = (const half_t *)q, g.K = (const half_t *)k, g.V = (const half_t *)v, g.O = (half_t *)out, g.starts = starts, g.kv_starts = kv_starts;
    g.q_rs = d.q_strides[0], g.q_hs = d.q_strides[1], g.o_rs = d.o_strides[0], g.o_hs = d.o_strides[1];
    g.k_rs = d.k_strides[0], g.k_hs = d.k_strides[1], g.v_rs = d.v_strides[0], g.v_hs = d.v_strides[1];
    g.batch = d.batch, g.kv_heads = d.kv_heads, g.group = d.heads / d.kv_heads, g.D = d.head_dim;
    g.rows = d.rows, g.kv_rows = d.kv_rows, g.max_rows = d.max_rows, g.max_keys = d.max_keys, g.causal = d.causal;
    ragged_scale(g, d.scale);
    return launch_ragged(g, false, workspace, workspace_bytes, stream);
}

} // namespace rt
