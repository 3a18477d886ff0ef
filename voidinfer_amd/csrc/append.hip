// append.hip — norms of queries and keys per head, their rotation, and the rows'
// keys and values written to the lanes' pages, in one pass (vi_norm_rotate_append).
//
// y = x / sqrt(mean(x^2) + eps) * w, then the first places turned by the row's
// angles, all in fp32 and rounded once to the cache's type.
//
// A head vector is read once and written once: the kernel is bound by those
// bytes.  Each thread holds two 16-byte chunks of one head, the two whose elements
// turn together (i and i + rotary/2) where the rotation is by halves, so the
// rotation needs no exchange; the mean square is summed in fp32 over the threads
// of a head, a power of two of them, by lane exchanges.
//
// 16,384 rows of 32 + 2 x 8 heads of 128 bf16 places (403 MB both ways): 102 to 106
// us, 3.9 TB/s against 4.8 of a plain copy; 8 rows 5.1 us and 136 rows 5.8 us, the
// look-ups of lane, page and angle one behind the other.  One head a thread: with
// two and four, whose look-ups are shared, the long case takes 112 to 114 us
// (fewer loads in flight a wave) and 8 rows 6.4 to 8.4.
#include "cache_rows.h"

namespace vi {
namespace {

constexpr int kAppendThreads = 256;

struct AppendArgs {
    vi_kv_cache cache;
    vi_lane_rows lanes;
    vi_head_rows q, k, v;
    vi_rotation rot;
    const void* q_weight;
    const void* k_weight;
    void* out;
    int64_t out_row, out_head;
    uint32_t* row_flags;
    float eps;
    int heads, pairs, group;   // pairs of chunks in a head; threads that share a head (a power of two >= pairs)
};

template <int DT> __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = Elem<DT>::decode(vec_bits<DT>(v, j));
}
template <int DT> __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = Elem<DT>::round(x[2 * j]) | (Elem<DT>::round(x[2 * j + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a) {
    const int per_block = kAppendThreads / a.group;
    const int total = a.heads + 2 * a.cache.kv_heads;
    const int64_t item = int64_t(blockIdx.x) * per_block + threadIdx.x / a.group;
    const int p = threadIdx.x % a.group;
    const int r = int(item / total), h = int(item % total);
    const bool live = r < a.lanes.rows && r < a.lanes.row_offsets[a.lanes.lanes];
    const bool work = live && p < a.pairs;
    const bool is_q = h < a.heads, is_v = h >= a.heads + a.cache.kv_heads;
    const int kv = is_q ? 0 : is_v ? h - a.heads - a.cache.kv_heads : h - a.heads;
    // chunk pair p: (p, p + rotary / 16) where the halves turn, then neighbours
    const int turning = a.rot.rotary_dim / 16;
    const int c0 = p < turning ? p : 2 * turning + 2 * (p - turning), c1 = p < turning ? p + turning : c0 + 1;

    float x0[8] = {}, x1[8] = {};
    uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
    if (work) {
        const vi_head_rows& s = is_q ? a.q : is_v ? a.v : a.k;
        const uint16_t* const in = static_cast<const uint16_t*>(s.data) + int64_t(r) * s.row_stride +
                                   int64_t(is_q ? h : kv) * s.head_stride;
        v0 = *reinterpret_cast<const uint4*>(in + 8 * c0);
        v1 = *reinterpret_cast<const uint4*>(in + 8 * c1);
    }
    int page = -1, place = 0;
    int64_t angle = 0;
    bool placed = false;
    if (live) {
        const int lane = lane_of_row(a.lanes.row_offsets, a.lanes.lanes, r);
        const int64_t index = int64_t(a.lanes.context[lane]) + (r - a.lanes.row_offsets[lane]);
        page = page_of(a.lanes, a.cache.pages, a.cache.page_size, lane, index);
        place = int(index & (a.cache.page_size - 1));
        angle = a.rot.positions ? int64_t(a.rot.positions[r]) : index;
        placed = page >= 0 && (a.rot.rotary_dim == 0 || (angle >= 0 && angle < a.rot.angle_rows));
    }
    if (!is_v) {
        unpack<DT>(v0, x0);
        unpack<DT>(v1, x1);
        const void* const weight = is_q ? a.q_weight : a.k_weight;
        if (weight) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf(x0[j], x0[j], s);
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf(x1[j], x1[j], s);
            for (int o = a.group >> 1; o; o >>= 1) s += __shfl_xor(s, o, kWave);
            const float inv = 1.0f / sqrtf(s / float(a.cache.head_dim) + a.eps);
            if (work) {
                float w0[8], w1[8];
                unpack<DT>(reinterpret_cast<const uint4*>(weight)[c0], w0);
                unpack<DT>(reinterpret_cast<const uint4*>(weight)[c1], w1);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x0[j] = x0[j] * inv * w0[j];
                    x1[j] = x1[j] * inv * w1[j];
                }
            }
        }
        if (work && placed && p < turning) {
            const int half = a.rot.rotary_dim / 2;
            const float* const cosines = a.rot.cosines + angle * half;
            const float* const sines = a.rot.sines + angle * half;
            if (a.rot.interleaved) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float ca = cosines[4 * c0 + j], sa = sines[4 * c0 + j];
                    const float cb = cosines[4 * c1 + j], sb = sines[4 * c1 + j];
                    const float u0 = x0[2 * j] * ca - x0[2 * j + 1] * sa, u1 = x0[2 * j] * sa + x0[2 * j + 1] * ca;
                    const float t0 = x1[2 * j] * cb - x1[2 * j + 1] * sb, t1 = x1[2 * j] * sb + x1[2 * j + 1] * cb;
                    x0[2 * j] = u0; x0[2 * j + 1] = u1;
                    x1[2 * j] = t0; x1[2 * j + 1] = t1;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float c = cosines[8 * c0 + j], s = sines[8 * c0 + j];
                    const float u = x0[j] * c - x1[j] * s, t = x0[j] * s + x1[j] * c;
                    x0[j] = u;
                    x1[j] = t;
                }
            }
        }
        if (!placed) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x0[j] = x1[j] = __builtin_nanf("");
        }
        v0 = pack<DT>(x0);
        v1 = pack<DT>(x1);
    }
    if (!work) return;
    if (a.row_flags && h == 0 && p == 0) a.row_flags[r] = placed ? 0u : uint32_t(VI_FLAG_ERROR);
    uint16_t* to;
    if (is_q) {
        to = static_cast<uint16_t*>(a.out) + int64_t(r) * a.out_row + int64_t(h) * a.out_head;
    } else {
        if (!placed) return;
        to = static_cast<uint16_t*>(is_v ? a.cache.values : a.cache.keys) + int64_t(page) * a.cache.page_stride +
             int64_t(kv) * a.cache.head_stride + int64_t(place) * a.cache.token_stride;
    }
    *reinterpret_cast<uint4*>(to + 8 * c0) = v0;
    *reinterpret_cast<uint4*>(to + 8 * c1) = v1;
}

}  // namespace

vi_status launch_append(const vi_kv_cache& cache, const vi_lane_rows& lanes, int heads, const vi_head_rows& q,
                        const vi_head_rows& k, const vi_head_rows& v, const void* q_weight, const void* k_weight,
                        float eps, const vi_rotation& rot, void* out, int64_t out_row, int64_t out_head,
                        uint32_t* row_flags, hipStream_t stream) {
    AppendArgs a{cache, lanes, q, k, v, rot, q_weight, k_weight, out, out_row, out_head, row_flags, eps, heads,
                 cache.head_dim / 16, 1};
    while (a.group < a.pairs) a.group <<= 1;
    const int64_t items = int64_t(lanes.rows) * (heads + 2 * int64_t(cache.kv_heads));
    const int64_t per = kAppendThreads / a.group, blocks = (items + per - 1) / per;
    if (blocks > 0x7fffffff) return VI_ERR_UNSUPPORTED;
    auto* kernel = cache.dtype == VI_BF16 ? append_kernel<VI_BF16> : append_kernel<VI_F16>;
    hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kAppendThreads), 0, stream, a);
    return launch_status();
}

}  // namespace vi
