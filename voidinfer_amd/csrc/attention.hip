// attention.hip — attention of the lanes' rows over their paged cache
// (vi_prefix_attention).
//
// One wave per (row, query head), one pass over the row's keys with a running
// maximum m and sum l per lane of the wave: each lane takes every 64th key whole
// and keeps its own m, l and weighted values in LDS, joined at the end.
#include "cache_rows.h"

namespace vi {
namespace {

struct AttnArgs {
    vi_kv_cache cache;
    vi_lane_rows lanes;
    vi_head_rows q;
    int heads, groups;
    float scale;
    const int32_t* group_offsets;
    const int32_t* prefix_lens;
    int max_rows, max_group_rows;
    const uint64_t* tree;
    void* out;
    int64_t out_row, out_head;
    float* lse;
};

template <int DT>
__global__ __launch_bounds__(64) void attention_row_kernel(AttnArgs a) {
    __shared__ float qs[512];
    __shared__ float acc[512];
    const int r = blockIdx.x / a.heads, h = blockIdx.x % a.heads, t = threadIdx.x, d = a.cache.head_dim;
    if (r >= a.lanes.row_offsets[a.lanes.lanes]) return;
    const int lane = lane_of_row(a.lanes.row_offsets, a.lanes.lanes, r);
    const int i = r - a.lanes.row_offsets[lane], rows = a.lanes.row_offsets[lane + 1] - a.lanes.row_offsets[lane];
    const int kv = h / (a.heads / a.cache.kv_heads);
    const int64_t context = a.lanes.context[lane];
    int first = lane, prefix = 0, group_rows = 0;
    for (int g = 0; g < a.groups; ++g)
        if (a.group_offsets[g] <= lane && lane < a.group_offsets[g + 1]) {
            first = a.group_offsets[g];
            prefix = a.prefix_lens[g];
            group_rows = a.lanes.row_offsets[a.group_offsets[g + 1]] - a.lanes.row_offsets[first];
        }
    const uint16_t* const q = static_cast<const uint16_t*>(a.q.data) + int64_t(r) * a.q.row_stride + int64_t(h) * a.q.head_stride;
    for (int e = t; e < d; e += 64) { qs[e] = Elem<DT>::decode(q[e]) * a.scale; acc[e] = 0.0f; }
    __syncthreads();
    const uint64_t seen = a.tree ? a.tree[r] : 0;
    float m = -kInfF, l = 0.0f;
    bool poison = i >= a.max_rows || (a.groups && group_rows > a.max_group_rows);
    for (int64_t k0 = 0; k0 < context + rows; k0 += 64) {
        const int64_t at = k0 + t, j = at - context;
        bool see = at < context + rows && (j < 0 || (a.tree ? j < 64 && (seen >> j & 1) : j <= i));
        float s = -kInfF;
        const uint16_t* vrow = nullptr;
        if (see) {
            const int page = page_of(a.lanes, a.cache.pages, a.cache.page_size, at < prefix ? first : lane, at);
            if (page < 0) {
                poison = true;
            } else {
                const int64_t o = int64_t(page) * a.cache.page_stride + int64_t(kv) * a.cache.head_stride +
                                  int64_t(at & (a.cache.page_size - 1)) * a.cache.token_stride;
                const uint16_t* const krow = static_cast<const uint16_t*>(a.cache.keys) + o;
                vrow = static_cast<const uint16_t*>(a.cache.values) + o;
                s = 0.0f;
                for (int e = 0; e < d; ++e) s = fmaf(qs[e], Elem<DT>::decode(krow[e]), s);
            }
        }
        float top = s;
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
        const float next = fmaxf(m, top);
        if (next == -kInfF) continue;
        const float shrink = expf(m - next), w = vrow ? expf(s - next) : 0.0f;
        float sum = w;
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, kWave);
        l = l * shrink + sum;
        m = next;
        for (int e = 0; e < d; ++e) {
            float x = vrow ? w * Elem<DT>::decode(vrow[e]) : 0.0f;
            for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, kWave);
            if (t == 0) acc[e] = acc[e] * shrink + x;
        }
    }
    if (ballot(poison)) l = m = __builtin_nanf("");
    __syncthreads();
    uint16_t* const out = static_cast<uint16_t*>(a.out) + int64_t(r) * a.out_row + int64_t(h) * a.out_head;
    for (int e = t; e < d; e += 64) out[e] = uint16_t(Elem<DT>::round(l == 0.0f ? 0.0f : acc[e] / l));
    if (a.lse && t == 0) a.lse[int64_t(r) * a.heads + h] = l == 0.0f ? -kInfF : m + logf(l);
}

}  // namespace

size_t attention_workspace(int rows, int heads, int kv_heads, int head_dim, int lanes, int groups, int max_rows,
                           int max_group_rows, int64_t max_own, int64_t max_prefix) {
    return 256;
}

vi_status launch_attention(const vi_kv_cache& cache, const vi_lane_rows& lanes, int heads, const vi_head_rows& q,
                           float scale, int groups, const int32_t* group_offsets, const int32_t* prefix_lens,
                           int max_rows, int max_group_rows, int64_t max_own, int64_t max_prefix,
                           const uint64_t* tree, void* out, int64_t out_row, int64_t out_head, float* lse, void* ws,
                           size_t ws_bytes, hipStream_t stream) {
    AttnArgs a{cache, lanes, q, heads, groups, scale, group_offsets, prefix_lens, max_rows, max_group_rows, tree, out,
               out_row, out_head, lse};
    const int64_t blocks = int64_t(lanes.rows) * heads;
    if (blocks > 0x7fffffff) return VI_ERR_UNSUPPORTED;
    auto* kernel = cache.dtype == VI_BF16 ? attention_row_kernel<VI_BF16> : attention_row_kernel<VI_F16>;
    hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(64), 0, stream, a);
    return launch_status();
}

}  // namespace vi
