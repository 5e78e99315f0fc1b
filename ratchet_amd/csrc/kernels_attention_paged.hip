// Attention over a key/value cache held in pages, up to 32 rows per head of keys (ragged.h): a step of one or a few tokens of every sequence.
//
//   out[m] = sum_j p_j v_j,  p = softmax_j(scale * q[m] . k_j);  row m = query row * group + head of the group
//
// What has to be done is to read the pages once, so the kernel is laid out around the loads: each of a workgroup's four (or eight) wavefronts takes 32 keys of 128 in turn, brings
// them into a part of LDS of its own, straight from memory, and waits for nobody else.  There is one block of keys and one of values: a wavefront asks for its next keys as soon as
// the scores are made, and for the values behind them when those are multiplied, so that 8 to 16 KB a wavefront are on their way at any time.
//   S^T = K Q^T and O^T += V^T P^T by v_mfma_f32_16x16x32_f16, as in kernels_attention_ragged.hip: a lane has four keys of 16 for one row, its probabilities are an operand as
//   they lie, and the values' comes transposed out of LDS.
// The work is the line of all 128 keys of all sequences and heads of keys; a workgroup takes an equal part of it, whatever the sequences' lengths, and so ends within a sequence.
// What it has of one that others share goes to the workspace, at most twice, and a second kernel joins the parts in a fixed order.  Lengths stay on the device.
//
// 32 sequences of up to 8192 keys, 8 heads of 128, one row of 32 heads, 684 MB: 110 us, 6.2 TB/s, as a copy of this kernel that only loads takes, and 4.7 in the join.  Small ones wait: 100 keys of
// 32 heads of 80 5.8 us, in a launch, three trips to memory one after another (lengths, pages, keys) and one step; 1024 keys 6.8 and 3.4 in the join.
#include "ragged.h"

#include <algorithm>

namespace rt {

constexpr int PS_KEYS = 128, PS_UNIT = 32; // of a workgroup's step, of a wavefront's
constexpr int ps_pitch(int ks) { return ks <= 4 ? 64 : 128; }
constexpr int ps_ring(int ks) { return 2 * PS_UNIT * ps_pitch(ks) * 2; } // bytes of a wavefront
typedef __fp16 ps_fp16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ constexpr int ps_waitcnt(int n) { return 0x0070 | (n & 0xF) | (((n >> 4) & 0x3) << 14); } // vmcnt(n) lgkmcnt(0)

// Everything of this wavefront's has arrived and been written, for the compiler too: loads into LDS behind this find nothing in their way.
__device__ __forceinline__ void ps_settle() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(ps_waitcnt(0));
    asm volatile("" ::: "memory");
}

// As rr_swizzle of the tiled kernel: rows four apart differ in the low bits, neighbours in the high ones.
template <int PITCH> __device__ __forceinline__ int ps_swizzle(int r) {
    return PITCH == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Steps of a sequence (at least one where it has rows: they are NaN), and of all up to a sequence.
struct PagedSeq {
    int first, rows, keys, steps;
    int off; // causal: row i sees keys up to i + off
};
__device__ __forceinline__ PagedSeq ps_seq(const RaggedArgs &g, int b) {
    PagedSeq s;
    int unused, all;
    const int at = min(b, g.batch - 1);
    s.rows = rg_rows(g, at, s.first), s.keys = rg_keys<true>(g, at, unused, all);
    s.off = all - rg_all_rows(g, at, s.first);
    s.steps = b < g.batch && s.rows > 0 ? max(1, (s.keys + PS_KEYS - 1) / PS_KEYS) : 0;
    return s;
}

// The place in the line at which workgroup i begins, and which workgroup has place c.
// (No more workgroups than places.)
__device__ __forceinline__ int ps_begin(int64_t i, int64_t total, int wgs) { return (int)(i * total / wgs); }
__device__ __forceinline__ int ps_owner(int64_t c, int64_t total, int wgs) { return (int)(((c + 1) * wgs + total - 1) / total) - 1; }

// KS: steps of 16 over head_dim (the last may be half).  NR: tiles of 16 rows.  NW: wavefronts; eight only with a head of keys each
template <int KS, int NR, int NW> __global__ __launch_bounds__(64 * NW, 2) void attention_paged_stream_kernel(RaggedArgs g, int whole) {
    constexpr int P = ps_pitch(KS), CPR = P / 8, KK = KS / 2, ODD = KS & 1, RPI = 64 / CPR, NI = PS_UNIT / RPI, NC = NI / 2; // (rows of a load instruction; instructions of a block, of 16 rows)
    constexpr int BLK = PS_UNIT * P; // halves of a block of keys, of values
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    half_t *const mine = (half_t *)(smem + wave * ps_ring(KS));  // this wavefront's [keys | values][32][P]
    float *const sums = (float *)(smem + NW * ps_ring(KS));       // [wavefront][row][2]

    // ---- where this workgroup begins and ends
    int b = 0, kh = 0, step = 0, todo, wgs = 0;
    int64_t total = 0, from = 0; // places in the line; that of this head of keys' first step
    PagedSeq seq;
    auto of_lane = [&](PagedSeq s, int l) {
        return PagedSeq{__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.rows, l), __builtin_amdgcn_readlane(s.keys, l), __builtin_amdgcn_readlane(s.steps, l),
                        __builtin_amdgcn_readlane(s.off, l)};
    };
    if (whole) { // a head of keys each
        b = blockIdx.x / g.kv_heads, kh = blockIdx.x - b * g.kv_heads;
        seq = of_lane(ps_seq(g, b), 0);
        todo = seq.steps;
    } else {
        const PagedSeq s0 = ps_seq(g, lane);
        total = rg_sum(s0.steps);
        for (int c = 64; c < g.batch; c += 64) total += rg_sum(ps_seq(g, c + lane).steps);
        total *= g.kv_heads;
        wgs = (int)min((int64_t)gridDim.x, total);
        if ((int)blockIdx.x >= wgs) return;
        const int begin = ps_begin(blockIdx.x, total, wgs);
        int at = begin;
        todo = ps_begin(blockIdx.x + 1, total, wgs) - at;
        PagedSeq s = s0;
        for (int c = 0;;) {
            const int upto = rg_scan(s.steps, lane), all = __builtin_amdgcn_readlane(upto, 63);
            if (at < all * g.kv_heads) { // (no step count passes 31 bits: host)
                const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto * g.kv_heads > at));
                seq = of_lane(s, l);
                at -= (__builtin_amdgcn_readlane(upto, l) - seq.steps) * g.kv_heads;
                b = c + l, kh = at / seq.steps, step = at - kh * seq.steps;
                break;
            }
            at -= all * g.kv_heads;
            c += 64;
            if (c >= g.batch) return; // (not reached: the place is in the line)
            s = ps_seq(g, c + lane);
        }
        from = begin - step;
    }
    b = __builtin_amdgcn_readfirstlane(b), kh = __builtin_amdgcn_readfirstlane(kh), step = __builtin_amdgcn_readfirstlane(step), todo = __builtin_amdgcn_readfirstlane(todo);
    if (todo <= 0) return;

    // Of the columns behind head_dim, which no load writes, the products read those of a last step that is half full: they are zeros.
    const bool half_step = g.D < 16 * KS;
    if (half_step) {
        for (int i = lane; i < ps_ring(KS) / 16; i += 64) ((uint4_t *)mine)[i] = uint4_t{0, 0, 0, 0};
        ps_settle();
    }
    // Loads: instruction i of 16 rows brings the rows RPI i ..; lane l the chunk l % CPR of row l / CPR, XOR-swizzled
    uint32_t from_page[NC]; // bytes
    uint64_t lanes[NC];     // those whose chunk is a part of the row
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int row = RPI * i + lane / CPR, c = 8 * ((lane % CPR) ^ ps_swizzle<P>(row));
        from_page[i] = 2u * (uint32_t)(row * g.D + c), lanes[i] = __builtin_amdgcn_ballot_w64(c < g.D);
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)mine;
    int koff[KK + ODD]; // the last of an odd number of steps by v_mfma_f32_16x16x16_f16: dimensions 16 KS - 16 + 4 fg ..
#pragma unroll
    for (int k = 0; k < KK; k++) koff[k] = fr * P + 8 * ((4 * k + fg) ^ ps_swizzle<P>(fr));
    if constexpr (ODD) koff[KK] = fr * P + 8 * ((4 * KK + (fg >> 1)) ^ ps_swizzle<P>(fr)) + 4 * (fg & 1);
    const int vrow = 4 * fg + (fr >> 2), vhalf = (fr & 3) >> 1;

    bool begun = false; // whether this is not the first head of keys of the workgroup
    while (todo > 0) {
        const int first = seq.first, n = seq.rows, len = seq.keys, all = seq.steps;
        const int upto = min(all, step + todo), rows = n * g.group, off = seq.off;
        auto sees = [&](int m) { return g.causal ? max(0, min(len, rg_query(g, m) + off + 1)) : len; };
        const int seen_all = sees(0), seen_any = sees(rows - 1);

        typedef __attribute__((address_space(4))) const int32_t *scalar_t; // read through the scalar cache
        const scalar_t table = (scalar_t)(uintptr_t)(g.table + b * g.table_stride);
        const int last_entry = max(0, len - 1) >> g.page_shift;
        const half_t *const K = g.K + (int64_t)kh * g.k_hs, *const V = g.V + (int64_t)kh * g.v_hs;
        int pages[2], at_keys; // of the next unit's 16 keys each; its first key
        auto look = [&](int j) __attribute__((always_inline)) {
            at_keys = j;
#pragma unroll
            for (int i = 0; i < 2; i++) pages[i] = table[min((j + 16 * i) >> g.page_shift, last_entry)];
        };
        int64_t where[2]; // of them in a pool, halves from the head's
        auto place = [&]() __attribute__((always_inline)) {
            uint32_t there = 3u;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const bool is = (uint32_t)pages[i] < (uint32_t)g.pages;
                if (!is) there &= ~(1u << i);
                where[i] = (int64_t)(is ? pages[i] : 0) * g.k_rs + (int64_t)(((at_keys + 16 * i) & ((1 << g.page_shift) - 1)) * g.D);
            }
            return there;
        };
        // (nt: a page is read once a step, and 32 sequences of up to 8192 keys take 116 us instead of 130 if it does not displace what is cached)
        auto issue = [&](const half_t *pool, uint32_t dst0) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const uint32_t dst = __builtin_amdgcn_readfirstlane(dst0 + 2u * RPI * i * P);
                // (every lane is active here, and is again)
                asm volatile("s_mov_b64 exec, %3\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt\n\ts_mov_b64 exec, -1" ::"s"(dst), "v"(from_page[i % NC]),
                             "s"(pool + where[i / NC]), "s"(lanes[i % NC])
                             : "m0", "memory");
            }
        };
        auto wait = [&](auto keep) __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(ps_waitcnt(decltype(keep)::value));
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        using All = std::integral_constant<int, 0>;
        using But = std::integral_constant<int, NI>;

        half8_t fq[NR][KK + 1]; // (without KK)
        half4_t ft[NR];
        int last[NR];
        float4_t acc[NR][KS];
        float c_run[NR], l_run[NR];
        bool coarse = false;
#pragma unroll
        for (int u = 0; u < NR; u++) {
            c_run[u] = -INFINITY, l_run[u] = 0.f;
#pragma unroll
            for (int d = 0; d < KS; d++) acc[u][d] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        auto values = [&](int d) __attribute__((always_inline)) { // dimensions 16 d ..; keys 4 fg .. and 16 + 4 fg ..
            typedef uint64_t u64x2_t __attribute__((ext_vector_type(2)));
            typedef __attribute__((address_space(3))) ps_fp16x4 *lds4;
            const half_t *p = mine + BLK + vrow * P + 8 * ((2 * d + vhalf) ^ ps_swizzle<P>(vrow)) + 4 * (fr & 1);
            const uint64_t v0 = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)p));
            const uint64_t v1 = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds4)(p + 16 * P)));
            return __builtin_bit_cast(half8_t, u64x2_t{v0, v1});
        };

        int j = step * PS_KEYS + PS_UNIT * wave; // this wavefront's keys
        const int j_end = min(upto * PS_KEYS, seen_any);
        if (j < j_end) {
            look(j);
            uint32_t there = place();
            issue(K, lds0), issue(V, lds0 + 2 * BLK);
#pragma unroll
            for (int u = 0; u < NR; u++) {
                const int m = min(16 * u + fr, rows - 1), qi = rg_query(g, m);
                last[u] = g.causal ? min(len - 1, qi + off) : len - 1;
                const half_t *q = g.Q + (int64_t)(first + qi) * g.q_rs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.q_hs;
#pragma unroll
                for (int k = 0; k < KK; k++) fq[u][k] = 32 * k + 8 * fg < g.D ? *(const half8_t *)(q + 32 * k + 8 * fg) : half8_t{};
                if constexpr (ODD) ft[u] = 32 * KK + 4 * fg < g.D ? *(const half4_t *)(q + 32 * KK + 4 * fg) : half4_t{};
            }
            constexpr int NEXT = NW * PS_UNIT; // keys to this wavefront's next
            bool more = j + NEXT < j_end;
            if (more) look(j + NEXT);
            if (g.sign != 1.f) {
                const half_t sign = (half_t)g.sign;
#pragma unroll
                for (int u = 0; u < NR; u++) {
#pragma unroll
                    for (int k = 0; k < KK; k++) fq[u][k] *= half8_t{sign, sign, sign, sign, sign, sign, sign, sign};
                    ft[u] *= half4_t{sign, sign, sign, sign};
                }
            }
            // awaited here: a first use in the loop would wait there, for these and with them for every load into LDS
#pragma unroll
            for (int u = 0; u < NR; u++) {
#pragma unroll
                for (int k = 0; k < KK; k++) asm volatile("" : "+v"(fq[u][k]));
                if constexpr (ODD) asm volatile("" : "+v"(ft[u]));
            }
            wait(But{});
            while (true) {
                // ---- scores
                // tail: a sum of its own.  With S as the third operand of the shorter instruction, heads of 72, 80 and 112 gave wrong scores: the compiler puts the two behind each other without a
                // wait, as it does (rightly) for two of one kind, and v_mfma_f32_16x16x32 seems not to hand its result on to an instruction of another length.  No other kernel here chains two kinds.
                float4_t S[NR][2], tail[NR][2];
#pragma unroll
                for (int u = 0; u < NR; u++) S[u][0] = S[u][1] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int k = 0; k < KK + ODD; k++) {
                        if (k < KK) {
                            const half8_t fk = *(const half8_t *)(mine + koff[k] + 16 * h * P);
#pragma unroll
                            for (int u = 0; u < NR; u++) S[u][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fk, fq[u][k], S[u][h], 0, 0, 0);
                        } else {
                            const half4_t fk = *(const half4_t *)(mine + koff[k] + 16 * h * P);
#pragma unroll
                            for (int u = 0; u < NR; u++) tail[u][h] = __builtin_amdgcn_mfma_f32_16x16x16f16(fk, ft[u], float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                        }
                    }
                if constexpr (ODD)
#pragma unroll
                    for (int u = 0; u < NR; u++) S[u][0] += tail[u][0], S[u][1] += tail[u][1];
                const uint32_t now = there;
                if (more) {
                    wait(But{}); // (of LDS: the keys have been read.  The values are not awaited: they are NI loads)
                    there = place();
                    issue(K, lds0);
                }
                // ---- softmax
                int left[NR];
#pragma unroll
                for (int u = 0; u < NR; u++) left[u] = last[u] - j - 4 * fg;
                const bool lean = j + PS_UNIT <= seen_all && now == 3u;
                auto sees_key = [&](int u, int e) { return 16 * (e >> 2) + (e & 3) <= left[u] && ((now >> (e >> 2)) & 1u); };
                half8_t fp[NR];
#pragma unroll
                for (int u = 0; u < NR; u++) {
                    if (!lean)
#pragma unroll
                        for (int e = 0; e < 8; e++) S[u][e >> 2][e & 3] = sees_key(u, e) ? S[u][e >> 2][e & 3] : -INFINITY;
                    float top = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, S[u][e >> 2][e & 3]);
                    top = rt_groups_max(top) * g.sc;
                    if (__builtin_amdgcn_ballot_w64(top - c_run[u] > RG_ABOVE)) {
                        const float c = fmaxf(c_run[u], top - RG_BELOW), alpha = c == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(c_run[u] - c);
                        c_run[u] = c;
                        l_run[u] *= alpha;
#pragma unroll
                        for (int d = 0; d < KS; d++) acc[u][d] *= alpha;
                        // (scores past 4096 are rounded before the reference is taken away: kernels_attention_ragged.hip)
                        coarse = coarse || __builtin_amdgcn_ballot_w64(c != -INFINITY && !(__builtin_fabsf(c) < 4096.f)) != 0;
                    }
                    const float sc = coarse ? 1.f : g.sc, c = c_run[u] == -INFINITY ? 0.f : c_run[u];
                    if (coarse)
#pragma unroll
                        for (int h = 0; h < 2; h++) S[u][h] *= g.sc;
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const half2_t p = {(half_t)__builtin_amdgcn_exp2f(fmaf(S[u][e >> 2][e & 3], sc, -c)), (half_t)__builtin_amdgcn_exp2f(fmaf(S[u][e >> 2][(e & 3) + 1], sc, -c))};
                        sum = __builtin_amdgcn_fdot2(p, half2_t{(half_t)1, (half_t)1}, sum, false);
                        fp[u][e] = p[0], fp[u][e + 1] = p[1];
                    }
                    l_run[u] += sum;
                }
                // ---- values
                if (more) wait(But{});
                else wait(All{});
                bool odd = false;
                if (!lean) { // a value that is not finite must not reach, as 0 * inf, the rows that do not see its key
                    float x = 0.f;
#pragma unroll
                    for (int d = 0; d < KS; d++) x = rg_odd(values(d), x);
                    odd = __builtin_amdgcn_ballot_w64(x != 0.f) != 0;
                }
                if (odd) {
                    half8_t vis[NR];
#pragma unroll
                    for (int u = 0; u < NR; u++)
#pragma unroll
                        for (int e = 0; e < 8; e++) vis[u][e] = __builtin_bit_cast(half_t, (uint16_t)(sees_key(u, e) ? 0x3C00 : 0));
                    asm volatile("" ::: "memory"); // (the values are read again)
#pragma unroll
                    for (int d = 0; d < KS; d++) {
                        half8_t v = values(d);
                        const half8_t code = rg_take_odd(v);
#pragma unroll
                        for (int u = 0; u < NR; u++) {
                            acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, fp[u], acc[u][d], 0, 0, 0);
                            const float4_t mark = __builtin_amdgcn_mfma_f32_16x16x32_f16(code, vis[u], float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                acc[u][d][i] += (int)mark[i] & 255 ? INFINITY : 0.f;
                                acc[u][d][i] += mark[i] >= 256.f ? -INFINITY : 0.f;
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < KS; d++) {
                        const half8_t v = values(d);
#pragma unroll
                        for (int u = 0; u < NR; u++) acc[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, fp[u], acc[u][d], 0, 0, 0);
                    }
                }
                if (!more) break;
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0): the values have been read
                asm volatile("" ::: "memory");
                issue(V, lds0 + 2 * BLK);
                j += NEXT;
                more = j + NEXT < j_end;
                if (more) look(j + NEXT);
                wait(But{}); // the keys
            }
        }
        // ---- the wavefronts' results: outputs where their blocks were, [tile][dimensions' tile][lane] four, references and sums
        float4_t *const rest = (float4_t *)mine;
#pragma unroll
        for (int u = 0; u < NR; u++) {
            const float l = rt_groups_sum(l_run[u]);
            if (fg == 0) *(float2_t *)(sums + 2 * (wave * 16 * NR + 16 * u + fr)) = float2_t{c_run[u], l};
#pragma unroll
            for (int d = 0; d < KS; d++) rest[(u * KS + d) * 64 + lane] = acc[u][d];
        }
        __syncthreads();
        const bool parted = step > 0 || upto < all; // others have the rest
        const int64_t slot = 2 * (int64_t)blockIdx.x + (begun ? 1 : 0);
        for (int e = t; e < NR * KS * 64; e += 64 * NW) {
            const int l = e & 63, ud = e >> 6, u = ud / KS, d = ud - u * KS, m = 16 * u + (l & 15), x = 16 * d + 4 * (l >> 4);
            if (m >= rows || x >= g.D) continue;
            float2_t ml[NW];
            float4_t o[NW];
#pragma unroll
            for (int w = 0; w < NW; w++) ml[w] = *(const float2_t *)(sums + 2 * (w * 16 * NR + m)), o[w] = *(const float4_t *)(smem + w * ps_ring(KS) + 16 * e);
            float top = ml[0][0];
#pragma unroll
            for (int w = 1; w < NW; w++) top = fmaxf(top, ml[w][0]);
            const float base = top == -INFINITY ? 0.f : top;
            float4_t y = {0.f, 0.f, 0.f, 0.f};
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float a = __builtin_amdgcn_exp2f(ml[w][0] - base);
                s = fmaf(ml[w][1], a, s);
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = fmaf(o[w][i], a, y[i]);
            }
            if (parted) {
                const int64_t at = slot * (g.max_rows * g.group) + m;
                *(float4_t *)(g.part_o + at * g.D + x) = y;
                if (x == 0) *(float2_t *)(g.part_ml + 2 * at) = float2_t{top, s};
            } else {
                const int qi = rg_query(g, m);
                half_t *const out = g.O + (int64_t)(first + qi) * g.o_rs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.o_hs + x;
                typedef half_t half4_u1 __attribute__((ext_vector_type(4), aligned(2)));
                const float inv = 1.f / s; // no visible key: 0 * inf, NaN
                *(half4_u1 *)out = half4_u1{(half_t)(y[0] * inv), (half_t)(y[1] * inv), (half_t)(y[2] * inv), (half_t)(y[3] * inv)};
            }
        }
        __syncthreads();
        if (half_step) { // the zeros again
            for (int i = lane; i < ps_ring(KS) / 16; i += 64) ((uint4_t *)mine)[i] = uint4_t{0, 0, 0, 0};
            ps_settle();
        }
        if (!whole && step == 0 && t == 0) { // for the join: who has parts of this head of keys
            int32_t *const o = g.owners + 2 * (b * g.kv_heads + kh);
            o[0] = 2 * (int)blockIdx.x + (begun ? 1 : 0), o[1] = ps_owner(from + all - 1, total, wgs);
        }
        todo -= upto - step, step = 0, begun = true, from += all;
        if (++kh == g.kv_heads && todo > 0) {
            kh = 0;
            do { // (empty sequences have no steps)
                if (++b >= g.batch) return; // (not reached: there are steps to do)
                seq = of_lane(ps_seq(g, b), 0);
            } while (seq.steps == 0);
        }
    }
}

// Joins the parts of a row (blockIdx.x: sequence, head of keys, row) in a fixed order: 32 threads have four columns each, 8 groups of them the parts.
__global__ __launch_bounds__(256) void attention_paged_join_kernel(RaggedArgs g) {
    __shared__ __attribute__((aligned(16))) float part[8][128], mls[8][2];
    const int t = threadIdx.x, per = g.max_rows * g.group;
    const int m = blockIdx.x % per, bk = blockIdx.x / per, b = bk / g.kv_heads, kh = bk - b * g.kv_heads;
    const int slot = g.owners[2 * bk], i1 = g.owners[2 * bk + 1], i0 = slot >> 1; // (not written for a sequence without rows)
    int first;
    const int n = rg_rows(g, b, first);
    if (m >= n * g.group || i0 == i1) return; // or it is written
    auto row_of = [&](int i) { return (int64_t)(i == i0 ? slot : 2 * i) * per + m; }; // workgroups behind the first begin with it
    const int c = t & 31, sg = t >> 5;
    const bool live = 4 * c < g.D;
    float top = -INFINITY, l = 0.f;
    float4_t y = {0.f, 0.f, 0.f, 0.f};
    for (int i = i0 + sg; i <= i1; i += 32) { // four parts at a time
        float2_t ml[4];
        float4_t v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t at = row_of(min(i + 8 * k, i1));
            ml[k] = *(const float2_t *)(g.part_ml + 2 * at), v[k] = *(const float4_t *)(g.part_o + at * g.D + (live ? 4 * c : 0));
            if (i + 8 * k > i1) ml[k] = float2_t{-INFINITY, 0.f}, v[k] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        const float now = fmaxf(fmaxf(top, fmaxf(ml[0][0], ml[1][0])), fmaxf(ml[2][0], ml[3][0])), base = now == -INFINITY ? 0.f : now;
        const float old = __builtin_amdgcn_exp2f(top - base);
        top = now, l *= old;
#pragma unroll
        for (int x = 0; x < 4; x++) y[x] *= old;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float a = __builtin_amdgcn_exp2f(ml[k][0] - base);
            l = fmaf(a, ml[k][1], l);
#pragma unroll
            for (int x = 0; x < 4; x++) y[x] = fmaf(a, v[k][x], y[x]);
        }
    }
    *(float4_t *)&part[sg][4 * c] = y;
    if (c == 0) mls[sg][0] = top, mls[sg][1] = l;
    __syncthreads();
    if (t < g.D) {
        float all = -INFINITY, sum = 0.f, s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) all = fmaxf(all, mls[k][0]);
        const float ref = all == -INFINITY ? 0.f : all;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float a = __builtin_amdgcn_exp2f(mls[k][0] - ref);
            sum = fmaf(part[k][t], a, sum), s = fmaf(mls[k][1], a, s);
        }
        const int qi = rg_query(g, m);
        g.O[(int64_t)(first + qi) * g.o_rs + (int64_t)(kh * g.group + (m - qi * g.group)) * g.o_hs + t] = (half_t)(sum / s);
    }
}

// How a call is run: on the kernels above where a head of keys has up to 32 rows, and then a head of keys a workgroup, or all in equal parts.  (8 sequences of 4096 keys, heads of 128, 32 and
// 33 of such rows: one row of as many heads on one of keys 13.9 and 18.2 us, and of 32 heads on 8, 8 and 9 rows, 33.5 and 33.3.)
struct PagedPlan {
    bool streams, whole;
    int wgs;
};
static PagedPlan ps_plan(const rt_attention_paged_desc &d) {
    const rt_paged_cache_desc &c = d.cache;
    const int64_t per = (int64_t)d.max_rows * (d.heads / c.kv_heads), heads = (int64_t)c.batch * c.kv_heads, steps = std::max(1, (d.max_keys + PS_KEYS - 1) / PS_KEYS);
    PagedPlan p{};
    p.streams = per <= 32 && heads <= 0xffffff && heads * steps < (int64_t(1) << 31) && heads * per < (int64_t(1) << 24);
    // A workgroup takes 5.8 us over a head of 100 keys and 0.8 more for each step, the join's launch 3.3 and more: few steps, or many heads, which keep the memory busy by themselves, are faster
    // without equal parts (us, in equal parts and a head each: 32 heads of 80, 8 steps 10.0 and 11.4; 96 of 96, 8 steps 15.6 and 13.1; 96 of 128, 12 steps 18.5 and 20.1; 128 of 128, 16 steps 24.1 and
    // 26.5; 256 of 128, 16 / 32 steps 39.6 / 67.7 and 35.0 / 66.6; 1024, 8 steps 71 and 60).
    p.whole = steps <= std::max<int64_t>(4, heads / 12);
    // Two workgroups to a compute unit where there is work for them: 32 x 8 heads, 16 steps; below, one, and half as many parts to join (96 heads of 96, 16 steps, 21.0 us with 512, 19.2 with 256).
    p.wgs = (int)std::min<int64_t>(heads * steps < 2048 ? 256 : 512, heads * steps);
    return p;
}

bool attention_paged_fits(const rt_attention_paged_desc &d) {
    if (d.cache.batch == 0 || d.heads == 0 || d.rows == 0) return true;
    return ragged_fits(d.cache.batch, d.cache.kv_heads, d.heads / d.cache.kv_heads, d.rows, d.max_rows);
}
uint64_t attention_paged_workspace_bytes(const rt_attention_paged_desc &d) {
    if (d.cache.batch == 0 || d.heads == 0 || d.rows == 0 || d.max_rows == 0) return 0;
    const PagedPlan p = ps_plan(d);
    if (!p.streams) return ragged_workspace_bytes(d.cache.batch, d.heads, d.cache.kv_heads, d.rows, d.max_rows, d.max_keys, d.cache.head_dim, d.causal);
    return p.whole ? 0 : (uint64_t)2 * p.wgs * d.max_rows * (d.heads / d.cache.kv_heads) * (d.cache.head_dim + 2) * sizeof(float) + (uint64_t)2 * d.cache.batch * d.cache.kv_heads * sizeof(int32_t);
}

template <int KS, int NR, int NW> static hipError_t launch_ps(const RaggedArgs &g, int whole, unsigned wgs, hipStream_t st) {
    constexpr size_t lds = NW * ps_ring(KS) + NW * 16 * NR * 2 * sizeof(float);
    if (const hipError_t e = ensure_lds_limit<&attention_paged_stream_kernel<KS, NR, NW>>(); e != hipSuccess) return e;
    hipLaunchKernelGGL((attention_paged_stream_kernel<KS, NR, NW>), dim3(wgs), dim3(64 * NW), lds, st, g, whole);
    return hipGetLastError();
}

hipError_t launch_attention_paged(const rt_attention_paged_desc &d, const void *q, const void *k_pool, const void *v_pool, const int32_t *table, const int32_t *lens,
                                  const int32_t *starts, void *out, void *workspace, uint64_t workspace_bytes, hipStream_t stream) {
    RaggedArgs g{};
    const rt_paged_cache_desc &c = d.cache;
    g.Q = (const half_t *)q, g.K = (const half_t *)k_pool, g.V = (const half_t *)v_pool, g.O = (half_t *)out, g.starts = starts, g.table = table, g.lens = lens;
    g.q_rs = d.q_strides[0], g.q_hs = d.q_strides[1], g.o_rs = d.o_strides[0], g.o_hs = d.o_strides[1];
    g.k_hs = g.v_hs = (int64_t)c.page_size * c.head_dim, g.k_rs = g.v_rs = g.k_hs * c.kv_heads; // a head's part of a page, a page
    g.table_stride = c.table_stride, g.pages = c.pages, g.page_shift = __builtin_ctz(c.page_size), g.table_width = c.table_width;
    g.batch = c.batch, g.kv_heads = c.kv_heads, g.group = d.heads / c.kv_heads, g.D = c.head_dim;
    g.rows = d.rows, g.max_rows = d.max_rows, g.max_keys = d.max_keys, g.causal = d.causal;
    if (c.pages == 0) g.max_keys = 0; // no page is there: no key
    ragged_scale(g, d.scale);
    PagedPlan p = ps_plan(d);
    if (!p.streams) return launch_ragged(g, true, workspace, workspace_bytes, stream);
    const int per = g.max_rows * g.group;
    const uint64_t need = attention_paged_workspace_bytes(d);
    if (!p.whole && workspace && workspace_bytes >= need && !((uintptr_t)workspace & 15u))
        g.part_o = (float *)workspace, g.part_ml = g.part_o + (uint64_t)2 * p.wgs * per * g.D, g.owners = (int32_t *)(g.part_ml + (uint64_t)4 * p.wgs * per);
    else
        p.whole = true;
    const unsigned wgs = p.whole ? (unsigned)(c.batch * c.kv_heads) : (unsigned)p.wgs;
    auto go = [&](auto ks) -> hipError_t {
        constexpr int KS = decltype(ks)::value;
        // Eight wavefronts, 133 KB of LDS, where a head of keys is a workgroup's, each has a compute unit and more than one step: half as many steps follow each other (us, with four and with eight:
        // 32 heads of 80, 512 keys 9.0 and 8.4; 96 of 96, 7 rows, 300 keys 8.2 and 7.5, 1000 keys 13.5 and 13.1; 256 of 128, 1024 keys 19.5 and 19.0).  One step leaves four of them idle (5.8 and 6.0),
        // and more heads than compute units do better with two workgroups of four to each (512 heads of 128, 300 keys 14.1 and 16.5; 1024, 1000 keys 62.1 and 67.3).
        if (p.whole && wgs <= 256 && g.max_keys > PS_KEYS) return per <= 16 ? launch_ps<KS, 1, 8>(g, 1, wgs, stream) : launch_ps<KS, 2, 8>(g, 1, wgs, stream);
        return per <= 16 ? launch_ps<KS, 1, 4>(g, p.whole, wgs, stream) : launch_ps<KS, 2, 4>(g, p.whole, wgs, stream);
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
    if (e != hipSuccess || p.whole) return e;
    hipLaunchKernelGGL(attention_paged_join_kernel, dim3((unsigned)(c.batch * c.kv_heads * per)), dim3(256), 0, stream, g);
    return hipGetLastError();
}

} // namespace rt
