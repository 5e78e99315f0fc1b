// Sequences of different lengths in one call: what the kernels of the paged cache and of packed prompts share.
#pragma once
#include "device_common.h"

namespace rt {

// Sequence b has the query rows starts[b] .. starts[b + 1] - 1 of one packed tensor (without `starts`: max_rows rows each).  Its keys lie in pages
// (table, lens), or packed like the queries (kv_starts; without it, where the queries lie).
struct RaggedArgs {
    const half_t *Q, *K, *V; // K, V: pools [pages, kv_heads, page, D], or packed rows
    half_t *O;
    float *part_o, *part_ml; // partial results of the shares of a row's keys
    const int32_t *starts, *kv_starts, *table, *lens;
    int64_t q_rs, q_hs, o_rs, o_hs, k_rs, k_hs, v_rs, v_hs, table_stride; // elements: rows, heads
    int batch, kv_heads, group, D, rows, kv_rows, max_rows, max_keys;
    int pages, page_shift, table_width;
    int causal, splits, tiles;
    int32_t *owners; // of the streaming kernel: for each sequence and head of keys the first workgroup that has a part (twice, and 1 where it is not its first) and the last
    float sc;  // |scale| log2(e), or 1 where the scale is 0
    float sign; // of the scale: the queries are multiplied by it (exactly)
    float per_group; // 1 / group
};

// m / group for m below 2^22 (group is at most 2^20): a multiple of 1 / group plus a half of that is further from a whole number than the product's error
__device__ __forceinline__ int rg_query(const RaggedArgs &g, int m) { return (int)(((float)m + 0.5f) * g.per_group); }

constexpr float kLog2eR = 1.4426950408889634f;
// The exponentials' reference is put this much, in base 2, below the maximum, and follows it where that is RG_ABOVE past it: outputs and sums are seldom rescaled, a probability
// (2^15 at most) is an f16, and those down to 2^-31 of the largest are not lost.
constexpr float RG_BELOW = 7.f, RG_ABOVE = 15.f;

// First query row and number of rows of a sequence, whatever `starts` holds inside the tensor.
__device__ __forceinline__ int rg_rows(const RaggedArgs &g, int b, int &first) {
    if (!g.starts) {
        first = b * g.max_rows;
        return g.max_rows;
    }
    const int a = min(max(g.starts[b], 0), g.rows), e = min(max(g.starts[b + 1], a), g.rows);
    first = a;
    return min(e - a, g.max_rows);
}
// Rows from `first` (rg_rows) to the sequence's end, those past max_rows or behind the tensor too: by them goes which keys a row sees.
__device__ __forceinline__ int rg_all_rows(const RaggedArgs &g, int b, int first) { return g.starts ? max(g.starts[b + 1], first) - first : g.max_rows; }
// First key and number of keys.  `all`: with those past max_keys or behind the tensor.  (all - rg_all_rows + a row + 1 is `all` at most: it fits 31 bits.)
template <bool PAGED> __device__ __forceinline__ int rg_keys(const RaggedArgs &g, int b, int &first, int &all) {
    if constexpr (PAGED) {
        first = 0, all = max(g.lens[b], 0);
        return min(all, g.max_keys);
    } else {
        const int32_t *s = g.kv_starts ? g.kv_starts : g.starts;
        int a = b * g.max_rows, e = a + g.max_rows;
        if (s) a = s[b], e = s[b + 1];
        a = min(max(a, 0), g.kv_rows), e = max(e, a);
        first = a, all = e - a;
        return min(min(e, g.kv_rows) - a, g.max_keys);
    }
}

template <int CTRL> __device__ __forceinline__ int rg_dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
template <typename OP> __device__ __forceinline__ int rg_reduce(int v, OP op) { // over the 64 lanes
    v = op(v, rg_dpp<0x128>(v)), v = op(v, rg_dpp<0x124>(v)), v = op(v, rg_dpp<0x122>(v)), v = op(v, rg_dpp<0x121>(v));
    const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = op((int)a[0], (int)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    return __builtin_amdgcn_readfirstlane(op((int)b[0], (int)b[1]));
}
__device__ __forceinline__ int rg_sum(int v) {
    return rg_reduce(v, [](int a, int b) { return a + b; });
}
// sum over the lanes up to this one
__device__ __forceinline__ int rg_scan(int v, int lane) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const int o = __shfl_up(v, s);
        if (lane >= s) v += o;
    }
    return v;
}
// The place-th lane (from 0) of those in `mask`.
__device__ __forceinline__ int rg_nth(uint64_t mask, int place, int lane) {
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    return __builtin_ctzll(__builtin_amdgcn_ballot_w64(((mask >> lane) & 1) && before == place));
}

// Every tile of TILE rows (query rows times heads that share a head of keys) of every sequence has a place in a line.  Tile t of a sequence comes before all tiles below t,
// so that with the causal flag the long ones come first; past 256 sequences the line goes by sequence instead.  -> whether there is such a place.
// `first`, `rows`: that sequence's.
template <int TILE> __device__ __forceinline__ bool rg_locate(const RaggedArgs &g, int place, int &b, int &tile, int &first, int &rows) {
    const int lane = threadIdx.x & 63;
    auto look = [&](int i, int &at, int &count) { // -> tiles
        count = rg_rows(g, min(i, g.batch - 1), at);
        return i < g.batch ? (count * g.group + TILE - 1) / TILE : 0;
    };
    if (g.batch <= 256) {
        int n[4], at[4], count[4], most = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            n[c] = at[c] = count[c] = 0;
            if (64 * c < g.batch) n[c] = look(64 * c + lane, at[c], count[c]);
            most = max(most, n[c]);
        }
        most = rg_reduce(most, [](int x, int y) { return max(x, y); });
        auto above = [&](int level) { // tiles of that number and up
            int s = 0;
#pragma unroll
            for (int c = 0; c < 4; c++) s += max(n[c] - level, 0);
            return rg_sum(s);
        };
        if (above(0) <= place) return false;
        int lo = 0, hi = most; // above(lo) > place >= above(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (above(mid) > place) lo = mid;
            else hi = mid;
        }
        place -= above(lo + 1);
        tile = lo;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint64_t mask = __builtin_amdgcn_ballot_w64(n[c] > lo);
            const int here = __builtin_popcountll(mask);
            if (place < here) {
                const int l = rg_nth(mask, place, lane);
                b = 64 * c + l, first = __builtin_amdgcn_readlane(at[c], l), rows = __builtin_amdgcn_readlane(count[c], l);
                return true;
            }
            place -= here;
        }
        return false;
    }
    for (int c = 0; c < g.batch; c += 64) {
        int from, count;
        const int n = look(c + lane, from, count), upto = rg_scan(n, lane), all = __builtin_amdgcn_readlane(upto, 63);
        if (place < all) {
            const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > place));
            b = c + at;
            tile = __builtin_amdgcn_readlane(upto, at) - 1 - place;
            first = __builtin_amdgcn_readlane(from, at), rows = __builtin_amdgcn_readlane(count, at);
            return true;
        }
        place -= all;
    }
    return false;
}

// The tiled kernel, for any number of rows (kernels_attention_ragged.hip): whether its grid holds a call, what workspace it asks for, the scale's part of
// the arguments, and the launch.
bool ragged_fits(int batch, int kv_heads, int group, int rows, int max_rows);
uint64_t ragged_workspace_bytes(int batch, int heads, int kv_heads, int rows, int max_rows, int max_keys, int head_dim, int causal);
void ragged_scale(RaggedArgs &g, float scale);
hipError_t launch_ragged(RaggedArgs &g, bool paged, void *workspace, uint64_t workspace_bytes, hipStream_t stream);

// Whether pairs of f16 are finite: the sum of their products with 0 is NaN where one is not.
__device__ __forceinline__ float rg_odd(half8_t v, float t) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) t = __builtin_amdgcn_fdot2(half2_t{v[e], v[e + 1]}, half2_t{(half_t)0, (half_t)0}, t, false);
    return t;
}

// Takes what is not finite out of v (0 in its place); -> 1 in the places of +inf, 256 of -inf, 257 of NaN, 0 else.
__device__ __forceinline__ half8_t rg_take_odd(half8_t &v) {
    uint4_t w = __builtin_bit_cast(uint4_t, v), code;
    auto spread = [](uint32_t top) { return top | (top - (top >> 15)); }; // bit 15 of a half to all of it
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t odd = spread(((w[i] & 0x7C007C00u) + 0x04000400u) & 0x80008000u);
        const uint32_t nan = spread((((w[i] & 0x03FF03FFu) + 0x03FF03FFu) & 0x04000400u) << 5);
        const uint32_t inf = 0x3C003C00u + ((w[i] & 0x80008000u) >> 2); // 1 and 256 as f16 differ by what is the sign bit moved down two
        code[i] = ((inf & ~nan) | (0x5C045C04u & nan)) & odd;
        w[i] &= ~odd;
    }
    v = __builtin_bit_cast(half8_t, w);
    return __builtin_bit_cast(half8_t, code);
}

} // namespace rt
