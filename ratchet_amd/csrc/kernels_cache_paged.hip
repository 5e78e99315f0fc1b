// The write of packed new rows into a key/value cache held in pages (ragged.h):
//   pool[table[b][p / page], h, p % page, :] = src[r, h, :],   b the sequence of row r, p = lens[b] - (its rows) + (r - starts[b]).
// A wavefront takes a row: it finds the row's sequence (64 starts at a time), its place, its page, and moves the row's heads of keys and values, 16 bytes
// of the pool a lane.  What has to be read and written is all that is moved: 11008 rows of 24 heads of 96 from f32, 304 MB, 66 us, 4.6 TB/s (a copy 5.1; loads and stores that leave the caches
// alone take as long).  32 rows of 8 heads of 128 4.2 us: three loads depend on one another before the first store.
#include "ragged.h"

namespace rt {

struct CachePagedArgs {
    half_t *pool[2];
    const void *src[2];
    const int32_t *starts, *table, *lens;
    int64_t s_rs, s_hs, table_stride;
    int batch, heads, D, rows, each, pages, page_shift, table_width, tensors;
};

template <typename T> __global__ __launch_bounds__(256) void cache_write_paged_kernel(CachePagedArgs g) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (r >= g.rows) return;
    int b;
    int64_t first, n;
    if (g.starts) { // sequences that end at or before this row
        b = 0;
        for (int c = 0; c < g.batch; c += 64) {
            const int i = c + lane;
            const int here = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < g.batch && g.starts[min(i, g.batch - 1) + 1] <= r));
            b += here;
            if (here < 64) break;
        }
        if (b >= g.batch) return; // behind the last
        first = g.starts[b], n = g.starts[b + 1] - first;
        if (r < first) return; // before the first
    } else {
        b = r / g.each, first = b * g.each, n = g.each;
    }
    const int64_t p = (int64_t)g.lens[b] - n + (r - first);
    const int64_t entry = p >> g.page_shift;
    if (p < 0 || entry >= g.table_width) return;
    const int page = g.table[b * g.table_stride + entry];
    if (page < 0 || page >= g.pages) return;
    const int per = g.D >> 3, count = g.heads * per * g.tensors; // groups of eight values
    const int slot = (int)(p & ((1 << g.page_shift) - 1));
    for (int i = lane; i < count; i += 64) {
        const int z = i >= g.heads * per, u = z ? i - g.heads * per : i, h = u / per, d = 8 * (u - h * per);
        const T *src = (const T *)g.src[z] + r * g.s_rs + h * g.s_hs + d;
        uint4_t raw;
        if constexpr (sizeof(T) == 2) {
            raw = *(const uint4_t *)src;
        } else {
            const float4_t lo = *(const float4_t *)src, hi = *(const float4_t *)(src + 4);
            raw = __builtin_bit_cast(uint4_t, half8_t{(half_t)lo[0], (half_t)lo[1], (half_t)lo[2], (half_t)lo[3], (half_t)hi[0], (half_t)hi[1], (half_t)hi[2], (half_t)hi[3]});
        }
        *(uint4_t *)(g.pool[z] + ((((int64_t)page * g.heads + h) << g.page_shift) + slot) * g.D + d) = raw;
    }
}

hipError_t launch_cache_write_paged(const rt_paged_cache_desc &d, int src_dtype, void *k_pool, const void *k_src, void *v_pool, const void *v_src, const int64_t *strides,
                                    const int32_t *table, const int32_t *lens, const int32_t *starts, int rows, hipStream_t stream) {
    CachePagedArgs g{};
    g.pool[0] = (half_t *)k_pool, g.pool[1] = (half_t *)v_pool, g.src[0] = k_src, g.src[1] = v_src;
    g.starts = starts, g.table = table, g.lens = lens;
    g.s_rs = strides[0], g.s_hs = strides[1], g.table_stride = d.table_stride;
    g.batch = d.batch, g.heads = d.kv_heads, g.D = d.head_dim, g.rows = rows, g.each = rows / d.batch;
    g.pages = d.pages, g.page_shift = __builtin_ctz(d.page_size), g.table_width = d.table_width, g.tensors = v_pool ? 2 : 1;
    const dim3 grid((unsigned)(((int64_t)rows + 3) / 4));
    if (src_dtype == RT_F32) hipLaunchKernelGGL((cache_write_paged_kernel<float>), grid, dim3(256), 0, stream, g);
    else hipLaunchKernelGGL((cache_write_paged_kernel<half_t>), grid, dim3(256), 0, stream, g);
    return hipGetLastError();
}

} // namespace rt
