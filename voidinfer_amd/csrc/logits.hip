// logits.hip — rows of logits rewritten by penalties, biases and grammar masks
// before a decision is taken over them (vi_process_logits).
//
// One workgroup per (row, slice of 8,192 tokens).  A token's penalty needs its
// number of occurrences, a bias the last entry that names it: both are rare in a
// slice, so each thread requests its logits first (they stay in registers),
// then the workgroup goes over the lane's lists and notes what falls into the
// slice in LDS: a bitmap of touched tokens and, for these only, a counter and a
// bias index.  The arrays are never cleared as a whole: a first pass over the lists
// sets the bits and zeroes the entries it will use, a second adds.  Vectors of
// eight tokens whose byte of the bitmap is zero go through unread and unrounded.
#include <algorithm>

#include "penalty_state.h"
#include "vi_device.h"
#include "vi_internal.h"

namespace vi {
namespace {

constexpr int kRuleThreads = 512;
constexpr int kRuleSlice = 8192;
constexpr int kRuleWords = kRuleSlice / 32;

struct RuleArgs {
    const void* logits;
    void* out;
    int64_t stride, out_stride;
    int rows, vocabulary, slices;
    vi_logit_rules r;
    PenaltyLayout layout;
    uint32_t* row_flags;
    int count_at, bias_at;   // LDS words: the counters, the bias indices
};

template <int DT> constexpr uint32_t kMasked = DT == VI_BF16 ? 0xff80ff80u : DT == VI_F16 ? 0xfc00fc00u : 0xff800000u;

__device__ __forceinline__ void store16(void* p, const uint4& v) {
    *static_cast<u32x4_any_t*>(p) = u32x4_t{v.x, v.y, v.z, v.w};
}

// Element j of a vector replaced.
template <int DT> __device__ __forceinline__ void set_bits(uint4& v, int j, uint32_t b) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (DT == VI_F32) {
        w[j] = b;
    } else {
        w[j >> 1] = (j & 1) ? (w[j >> 1] & 0xffffu) | (b << 16) : (w[j >> 1] & 0xffff0000u) | b;
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
}

// The vector's elements whose mask bit is clear become -Inf.
template <int DT> __device__ __forceinline__ void apply_mask(uint4& v, uint32_t allowed) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t keep;
        if constexpr (DT == VI_F32) {
            keep = 0u - (allowed >> i & 1u);
        } else {
            keep = ((0u - (allowed >> (2 * i) & 1u)) & 0xffffu) | ((0u - (allowed >> (2 * i + 1) & 1u)) << 16);
        }
        w[i] = (w[i] & keep) | (kMasked<DT> & ~keep);
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
}

// The penalties of vi_row_params in fp32, one rounding an operation
// (penalize_bits without its last rounding: a bias may follow).
__device__ __forceinline__ float penalize_value(float y, uint32_t count, const vi_row_params& p) {
#pragma clang fp contract(off)
    if (p.repetition_penalty != 1.0f) y = (y > 0.0f) ? y / p.repetition_penalty : y * p.repetition_penalty;
    if (p.frequency_penalty != 0.0f) {
        const float t = p.frequency_penalty * float(count);
        y = y - t;
    }
    if (p.presence_penalty != 0.0f) y = y - p.presence_penalty;
    return y;
}

template <int DT>
__global__ __launch_bounds__(kRuleThreads) void rules_kernel(RuleArgs a) {
    constexpr int kPer = Elem<DT>::kPerVec, kVecs = kRuleSlice / (kRuleThreads * kPer);
    using Bits = typename Elem<DT>::Bits;
    extern __shared__ uint32_t lds[];
    uint32_t* const seen = lds;                   // tokens with an occurrence
    uint32_t* const biased = lds + kRuleWords;    // tokens with a bias
    uint32_t* const count = lds + a.count_at;
    uint32_t* const bias = lds + a.bias_at;

    const int tid = threadIdx.x, row = int(blockIdx.x / unsigned(a.slices)), slice = int(blockIdx.x % unsigned(a.slices));
    const int first = slice * kRuleSlice, n = min(kRuleSlice, a.vocabulary - first);
    const vi_logit_rules& r = a.r;
    const Bits* const in = static_cast<const Bits*>(a.logits) + int64_t(row) * a.stride + first;
    Bits* const out = static_cast<Bits*>(a.out) + int64_t(row) * a.out_stride + first;

    const int lane = r.row_lanes ? r.row_lanes[row] : row;
    const int mask = r.mask_index ? r.mask_index[row] : -1;
    bool failed = lane < 0 || lane >= r.lanes || mask >= r.masks;
    uint32_t flags = failed ? uint32_t(VI_FLAG_ERROR) : 0u;

    vi_row_params p{};
    bool penalties = false;
    if (!failed && r.params) {
        p = r.params[lane];
        penalties = penalties_active(p) && (r.histories || r.states || r.extra);
    }
    const unsigned char* state = nullptr;
    if (penalties && r.states) {
        state = static_cast<const unsigned char*>(r.states) + size_t(lane) * a.layout.lane_bytes;
        const uint32_t f = reinterpret_cast<const PenaltyHeader*>(state)->flags;
        flags |= f;
        if (f & uint32_t(VI_FLAG_ERROR)) failed = true;
    }
    const bool biases = !failed && r.bias_ids;
    penalties = penalties && !failed;

    // the thread's logits and mask bits: a masked vector's logits are not read
    uint4 v[kVecs];
    uint32_t allowed[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int t = (k * kRuleThreads + tid) * kPer;
        allowed[k] = failed ? 0u : (1u << kPer) - 1u;
        if (!failed && mask >= 0 && t < n) {
            const uint32_t w = r.mask_words[int64_t(mask) * r.mask_stride + ((first + t) >> 5)];
            allowed[k] &= w >> (t & 31);
        }
    }
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int t = (k * kRuleThreads + tid) * kPer;
        v[k] = make_uint4(0, 0, 0, 0);
        if (t + kPer <= n) {
            if (allowed[k]) v[k] = load16(in + t);
        } else if (t < n) {
            for (int j = 0; j < kPer; ++j)
                if (t + j < n) set_bits<DT>(v[k], j, load_bits<DT>(in, t + j));
        }
    }

    if (penalties || biases) {
        for (int i = tid; i < 2 * kRuleWords; i += kRuleThreads) lds[i] = 0u;
        __syncthreads();
        int64_t hb = 0, he = 0, eb = 0, ee = 0, bb = 0, be = 0;
        if (penalties && r.histories) { hb = r.history_offsets[lane]; he = r.history_offsets[lane + 1]; }
        if (penalties && r.extra) { eb = r.extra_offsets[row]; ee = r.extra_offsets[row + 1]; }
        if (biases) { bb = r.bias_offsets[lane]; be = r.bias_offsets[lane + 1]; }
        const uint32_t* const present = state ? reinterpret_cast<const uint32_t*>(state + a.layout.off_b1) : nullptr;
        const uint2* const table = state ? reinterpret_cast<const uint2*>(state + a.layout.off_hash) : nullptr;
        const int words = (n + 31) / 32;
        bool bad = false;
        auto mark = [&](const int32_t* list, int64_t b, int64_t e, uint32_t* bits, uint32_t* value) {
            for (int64_t i = b + tid; i < e; i += kRuleThreads) {
                const int t = list[i] - first;
                bad |= uint32_t(list[i]) >= uint32_t(a.vocabulary);
                if (uint32_t(t) < uint32_t(n)) {
                    atomicOr(&bits[t >> 5], 1u << (t & 31));
                    value[t] = 0u;
                }
            }
        };
        uint32_t mine = 0u;
        if (present && tid < words) {
            mine = present[(first >> 5) + tid];
            if (mine) atomicOr(&seen[tid], mine);
            for (uint32_t m = mine; m; m &= m - 1u) count[tid * 32 + __builtin_ctz(m)] = 0u;
        }
        mark(r.histories, hb, he, seen, count);
        mark(r.extra, eb, ee, seen, count);
        mark(r.bias_ids, bb, be, biased, bias);
        __syncthreads();
        for (uint32_t m = mine; m; m &= m - 1u) {
            const int t = tid * 32 + __builtin_ctz(m);
            atomicAdd(&count[t], hash_count(table, a.layout.shift, a.layout.slots, first + t));
        }
        auto add = [&](const int32_t* list, int64_t b, int64_t e) {
            for (int64_t i = b + tid; i < e; i += kRuleThreads) {
                const int t = list[i] - first;
                if (uint32_t(t) < uint32_t(n)) atomicAdd(&count[t], 1u);
            }
        };
        add(r.histories, hb, he);
        add(r.extra, eb, ee);
        for (int64_t i = bb + tid; i < be; i += kRuleThreads) {
            const int t = r.bias_ids[i] - first;
            if (uint32_t(t) < uint32_t(n)) atomicMax(&bias[t], uint32_t(i - bb));   // the last entry of a token
        }
        if (__syncthreads_or(bad)) flags |= uint32_t(VI_FLAG_BAD_HISTORY);
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int t = (k * kRuleThreads + tid) * kPer;
            if (t >= n) continue;
            constexpr uint32_t kAll = (1u << kPer) - 1u;
            const uint32_t s = seen[t >> 5] >> (t & 31) & kAll & allowed[k];
            const uint32_t b = biased[t >> 5] >> (t & 31) & kAll & allowed[k];
            if (!(s | b)) continue;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                if (!((s | b) >> j & 1u)) continue;
                float y = Elem<DT>::decode(vec_bits<DT>(v[k], j));
                if (s >> j & 1u) y = penalize_value(y, count[t + j], p);
                if (b >> j & 1u) y = y + r.bias_values[bb + bias[t + j]];
                set_bits<DT>(v[k], j, Elem<DT>::round(y));
            }
        }
    }
    if (a.row_flags && slice == 0 && tid == 0) a.row_flags[row] = flags;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int t = (k * kRuleThreads + tid) * kPer;
        apply_mask<DT>(v[k], allowed[k]);
        if (t + kPer <= n) {
            store16(out + t, v[k]);
        } else if (t < n) {
            for (int j = 0; j < kPer; ++j)
                if (t + j < n) out[t + j] = Bits(vec_bits<DT>(v[k], j));
        }
    }
}

}  // namespace

vi_status launch_rules(const void* logits, int dtype, int rows, int vocabulary, int64_t stride,
                       const vi_logit_rules& rules, void* out, int64_t out_stride, uint32_t* row_flags,
                       hipStream_t stream) {
    RuleArgs a{};
    a.logits = logits; a.out = out; a.stride = stride; a.out_stride = out_stride;
    a.rows = rows; a.vocabulary = vocabulary; a.slices = (vocabulary + kRuleSlice - 1) / kRuleSlice;
    a.r = rules; a.row_flags = row_flags;
    if (rules.states) a.layout = penalty_layout(vocabulary, rules.slots);
    size_t words = 2 * kRuleWords;
    a.count_at = int(words);
    if (rules.params && (rules.histories || rules.states || rules.extra)) words += kRuleSlice;
    a.bias_at = int(words);
    if (rules.bias_ids) words += kRuleSlice;
    const int64_t blocks = int64_t(rows) * a.slices;
    if (blocks > 0x7fffffff) return VI_ERR_UNSUPPORTED;
    auto* kernel = dtype == VI_BF16 ? rules_kernel<VI_BF16> : dtype == VI_F16 ? rules_kernel<VI_F16> : rules_kernel<VI_F32>;
    hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kRuleThreads), words * 4, stream, a);
    return launch_status();
}

}  // namespace vi
