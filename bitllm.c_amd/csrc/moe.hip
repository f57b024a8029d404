// moe.hip -- routing to experts: the choice from a router's logits, pairs sorted by expert, the weighted sum of the experts' rows
// (eif_hip_moe.h).
#include "hip_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>

#include "../../include/eif_hip_moe.h"

namespace {

constexpr int kMaxExperts = 4096, kMaxTop = 64, kMaxGroups = 64, kMaxPairs = 1 << 30;
constexpr int kMaxTokens = 1 << 25;            // of a choice: 64 threads each, and a launch holds fewer than 2^32
constexpr int kLaunchBlocks = (1 << 24) - 1;   // of 256 threads

inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// LDS that one wave writes and reads by itself: in order in the hardware, so that only the compiler has to be told.
EIF_DEV void wave_lds_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---- the choice ----

struct RouteArgs {
    const void *logits;
    const float *bias;
    int32_t *ids;
    float *weights;
    int64_t ldl;
    int type, tokens, experts, top, score, groups, kept, best, renormalise;
    int group_size;
    uint32_t group_magic;   // e / group_size = (e * group_magic) >> 32 for e < 4096 and group_size > 1
    float scale;
};

template <int LX>
EIF_DEV double xlane_d(double v)
{
    const float lo = xlane<LX>(__int_as_float(__double2loint(v))), hi = xlane<LX>(__int_as_float(__double2hiint(v)));
    return __hiloint2double(__float_as_int(hi), __float_as_int(lo));
}
template <int LX>
EIF_DEV float xlane_of(float v) { return xlane<LX>(v); }
template <int LX>
EIF_DEV double xlane_of(double v) { return xlane_d<LX>(v); }

// f over the lanes l ^ 1, ^ 2, .. of a group of LPT lanes.
template <int LPT, typename F>
EIF_DEV void butterfly(F f)
{
    f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 4>{});
    f(std::integral_constant<int, 8>{});
    if constexpr (LPT == 64) {
        f(std::integral_constant<int, 16>{});
        f(std::integral_constant<int, 32>{});
    }
}
template <int LPT, typename V>
EIF_DEV V lanes_max(V v)
{
    butterfly<LPT>([&](auto x) { v = fmax(v, xlane_of<decltype(x)::value>(v)); });
    return v;
}
template <int LPT, typename V>
EIF_DEV V lanes_sum(V v)
{
    butterfly<LPT>([&](auto x) { v += xlane_of<decltype(x)::value>(v); });
    return v;
}

EIF_DEV float logit_at(const RouteArgs &a, int64_t i)
{
    const float l = a.type == EIF_HIP_F32   ? static_cast<const float *>(a.logits)[i]
                    : a.type == EIF_HIP_F16 ? __half2float(static_cast<const __half *>(a.logits)[i])
                                            : __bfloat162float(static_cast<const __hip_bfloat16 *>(a.logits)[i]);
    return l > -INFINITY ? fminf(l, 3.402823466e+38f) : -INFINITY;   // NaN and -inf: shut out
}

// LPT lanes a token, lane `sub` of them has experts sub, sub + LPT, .. (VPL of them). KEY is what experts are compared by: their
// logits (float), or score plus bias (double; experts of equal scores in 32 bits can differ in 64, and which of them is chosen
// changes the token's result by a whole expert). The choice takes the largest top_k times over: each lane's best, the best of the lanes.
template <typename KEY, int LPT, int VPL>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a)
{
    extern __shared__ double lds[];
    constexpr int per_wave = 64 / LPT;
    constexpr bool wide = sizeof(KEY) == 8;
    const KEY none = -INFINITY;
    const int lane = threadIdx.x & 63, sub = lane % LPT, wave = threadIdx.x >> 6;
    const int mine = wave * per_wave + lane / LPT;   // of the workgroup's tokens
    const int64_t token = (int64_t)blockIdx.x * (blockDim.x / LPT) + mine;
    const bool live = token < a.tokens;
    const int64_t row = (live ? token : a.tokens - 1) * a.ldl;

    KEY by[VPL];
    float m = 0.0f, z = 0.0f;   // softmax: largest logit, sum of e^(l - m)
    double md = 0.0, zd = 0.0;
    {
        float l[VPL];
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = i * LPT + sub;
            l[i] = e < a.experts ? logit_at(a, row + e) : -INFINITY;
        }
        if (a.score == EIF_HIP_SCORE_SOFTMAX && (wide || !a.renormalise)) {
            m = l[0];
#pragma unroll
            for (int i = 1; i < VPL; ++i) m = fmaxf(m, l[i]);
            m = lanes_max<LPT>(m);
            if (m == -INFINITY) m = 0.0f;
            md = m;
        }
        if constexpr (wide) {
            double p[VPL];
            if (a.score == EIF_HIP_SCORE_SOFTMAX) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) {
                    p[i] = exp((double)l[i] - md);   // e^-inf = 0 where shut out
                    zd += p[i];
                }
                zd = lanes_sum<LPT>(zd);
#pragma unroll
                for (int i = 0; i < VPL; ++i) p[i] /= zd;
            } else {
#pragma unroll
                for (int i = 0; i < VPL; ++i) p[i] = 1.0 / (1.0 + exp(-(double)l[i]));
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = i * LPT + sub;
                const double b = a.bias && e < a.experts ? (double)a.bias[e] : 0.0;
                const bool open = l[i] > -INFINITY && b > -INFINITY;
                p[i] = open ? p[i] + b : none;
                by[i] = !open ? none : a.bias ? p[i] : (double)l[i];
                if (a.groups > 1 && e < a.experts) lds[mine * (a.experts + a.groups) + e] = p[i];
            }
        } else {
            if (a.score == EIF_HIP_SCORE_SOFTMAX && !a.renormalise) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) z += expf(l[i] - m);
                zd = lanes_sum<LPT>(z);
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                by[i] = l[i];
                const int e = i * LPT + sub;
                if (a.groups > 1 && e < a.experts) reinterpret_cast<KEY *>(lds)[mine * (a.experts + a.groups) + e] = l[i];
            }
        }
    }

    if (a.groups > 1) {
        KEY *val = reinterpret_cast<KEY *>(lds) + mine * (a.experts + a.groups), *worth = val + a.experts;
        wave_lds_order();
        for (int g = sub; g < a.groups; g += LPT) {
            KEY b1 = none, b2 = none;
            int at = g % a.group_size;   // lanes start at different experts of their groups: different LDS banks
            for (int j = 0; j < a.group_size; ++j) {
                const KEY v = val[g * a.group_size + at];
                at = at + 1 == a.group_size ? 0 : at + 1;
                if (v > b1) {
                    b2 = b1;
                    b1 = v;
                } else if (v > b2) {
                    b2 = v;
                }
            }
            worth[g] = a.best == 2 && b2 > none ? b1 + b2 : b1;
        }
        wave_lds_order();
        uint64_t keep = 0;
        for (int g0 = 0; g0 < a.groups; g0 += LPT) {
            const int g = g0 + sub;
            int better = a.kept;
            if (g < a.groups) {
                const KEY w = worth[g];
                better = 0;
                for (int h = 0; h < a.groups; ++h) better += worth[h] > w || (worth[h] == w && h < g);
            }
            const uint64_t bits = __ballot(better < a.kept);
            keep |= LPT == 64 ? bits : ((bits >> (lane & 48)) & 0xffff) << g0;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const uint32_t e = i * LPT + sub, g = a.group_size == 1 ? e : __umulhi(e, a.group_magic);
            if (!((keep >> (g & 63)) & 1)) by[i] = none;
        }
    }

    int chosen = -1;   // lane k: the token's k-th expert
    KEY value = none;
    for (int k = 0; k < a.top; ++k) {
        KEY best = none;
        int e = INT32_MAX;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            if (by[i] > best) {
                best = by[i];
                e = i * LPT + sub;
            }
        }
        butterfly<LPT>([&](auto x) {
            const KEY ob = xlane_of<decltype(x)::value>(best);
            const int oe = __float_as_int(xlane<decltype(x)::value>(__int_as_float(e)));
            if (ob > best || (ob == best && oe < e)) {
                best = ob;
                e = oe;
            }
        });
        if (sub == k) {
            chosen = e == INT32_MAX ? -1 : e;
            value = best;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) by[i] = i * LPT + sub == e ? none : by[i];
    }

    // the weights, a lane each, in 64 bits
    const bool there = chosen >= 0;
    double w = 0.0;
    const double l = there ? (wide ? (double)logit_at(a, row + chosen) : (double)value) : -INFINITY;
    if (a.score == EIF_HIP_SCORE_SOFTMAX) {
        if (a.renormalise) md = lanes_max<LPT>(l);
        w = there ? exp(l - md) : 0.0;
        if (a.renormalise) zd = lanes_sum<LPT>(w);
    } else {
        w = there ? 1.0 / (1.0 + exp(-l)) : 0.0;
        zd = a.renormalise ? lanes_sum<LPT>(w) : 1.0;
    }
    if (live && sub < a.top) {
        a.ids[token * a.top + sub] = chosen;
        a.weights[token * a.top + sub] = w > 0.0 ? (float)(w / zd * (double)a.scale) : 0.0f;
    }
}

// ---- pairs by expert ----

constexpr int kSortBlocks = 256;      // of a sort in two launches, at most: one a CU
constexpr int kSortAlone = 8192;      // pairs that one workgroup sorts in one launch
constexpr int kSortStep = 4096;       // pairs of a workgroup at least, in two launches

// Waves of a placing workgroup: each has a counter of every expert in LDS, 64 KB in all.
int sort_waves(int experts) { return experts > 2048 ? 2 : experts > 1024 ? 4 : experts > 512 ? 8 : 16; }
// Pairs of a workgroup, whole steps of its waves, and how many workgroups that takes.
int sort_share(int64_t pairs)
{
    const int64_t per = std::max<int64_t>(kSortStep, (pairs + kSortBlocks - 1) / kSortBlocks);
    return (int)((per + 1023) / 1024 * 1024);
}
int sort_blocks(int64_t pairs) { return pairs <= kSortAlone ? 1 : (int)((pairs + sort_share(pairs) - 1) / sort_share(pairs)); }

__global__ __launch_bounds__(1024) void sort_count_kernel(const int32_t *ids, int pairs, int share, int experts, int32_t *counts)
{
    extern __shared__ int32_t cnt[];
    for (int e = threadIdx.x; e < experts; e += blockDim.x) cnt[e] = 0;
    __syncthreads();
    const int lo = blockIdx.x * share, hi = min(pairs - lo, share);
    for (int i = threadIdx.x; i < hi; i += blockDim.x) {
        const int id = ids[lo + i];
        if ((unsigned)id < (unsigned)experts) atomicAdd(&cnt[id], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[blockIdx.x * experts + e] = cnt[e];
}

// Lanes of the wave that have this lane's id; none where `live` is false.
EIF_DEV uint64_t same_id(int id, bool live, int bits)
{
    uint64_t m = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const bool one = (id >> b) & 1;
        const uint64_t q = __ballot(one);
        m &= one ? q : ~q;
    }
    return live ? m : 0;
}

// A workgroup places the pairs [blockIdx share, + share): a pair's place is the pairs of lower experts, those of its expert in
// workgroups, waves and steps before, and in the lanes before. Each wave has a run of the pairs in order, and counters of its own.
__global__ __launch_bounds__(1024) void sort_place_kernel(const int32_t *ids, int pairs, int share, int experts, int bits, int top,
                                                          const int32_t *counts, int blocks, int32_t *offsets, int32_t *row, int32_t *slot)
{
    extern __shared__ int32_t cnt[];   // [waves][experts], then the sums [experts] and of the waves [16]
    const int threads = blockDim.x, waves = threads >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int32_t *sums = cnt + waves * experts, *part = sums + experts;
    int32_t *own = cnt + wave * experts;
    const int lo = blockIdx.x * share, n = min(pairs - lo, share), run = (n + waves * 64 - 1) / (waves * 64) * 64;
    for (int i = threadIdx.x; i < waves * experts; i += threads) cnt[i] = 0;
    __syncthreads();
    const int from = min(wave * run, n), to = min(from + run, n);
    for (int i = from + lane; i < to; i += 64) {
        const int id = ids[lo + i];
        if ((unsigned)id < (unsigned)experts) atomicAdd(&own[id], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += threads) {
        int before = 0, all = 0;
        if (blocks > 1) {
            for (int b = 0; b < blocks; ++b) {
                const int c = counts[b * experts + e];
                before += b < (int)blockIdx.x ? c : 0;
                all += c;
            }
        }
        for (int w = 0; w < waves; ++w) {
            const int c = cnt[w * experts + e];
            cnt[w * experts + e] = before;
            before += c;
        }
        sums[e] = blocks > 1 ? all : before;
    }
    __syncthreads();
    // exclusive sums over the experts: each thread's run of them, the wave's, the workgroup's
    const int each = (experts + threads - 1) / threads, first = min((int)threadIdx.x * each, experts), last = min(first + each, experts);
    int mine = 0;
    for (int e = first; e < last; ++e) mine += sums[e];
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(upto, d, 64);
        upto += lane >= d ? o : 0;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int at = upto - mine;
    for (int w = 0; w < wave; ++w) at += part[w];
    for (int e = first; e < last; ++e) {
        const int c = sums[e];
        sums[e] = at;
        if (blockIdx.x == 0) offsets[e] = at;
        at += c;
        if (blockIdx.x == 0 && e == experts - 1) offsets[experts] = at;
    }
    __syncthreads();
    for (int i = from; i < to; i += 64) {
        const int p = lo + i + lane;
        const int id = i + lane < to ? ids[p] : -1;
        const bool live = (unsigned)id < (unsigned)experts;
        const uint64_t same = same_id(id, live, bits);
        int place = -1;
        if (live) {
            place = sums[id] + own[id] + __popcll(same & ((1ull << lane) - 1));
            row[place] = p / top;
        }
        if (i + lane < to) slot[p] = place;
        wave_lds_order();
        if (live && (same >> lane) == 1) own[id] += __popcll(same);   // the last of the lanes that share an id
        wave_lds_order();
    }
}

// ---- the experts' rows together ----

template <typename T>
EIF_DEV T from_f32(float v);
template <>
EIF_DEV float from_f32<float>(float v) { return v; }
template <>
EIF_DEV __half from_f32<__half>(float v) { return __float2half(v); }
template <>
EIF_DEV __hip_bfloat16 from_f32<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

struct CombineArgs {
    const float *y, *weights, *add;
    const int32_t *slot;
    void *out;
    int64_t ldy, lda, ldo;
    int rows, tokens, top, dim;
    int cols, chunks, log_cols;   // threads of a token in a workgroup (2^log_cols of them), and workgroups of a token's columns
};

// A thread has V adjacent columns of a token.
template <typename T, int V>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a)
{
    const int64_t block = blockIdx.x / a.chunks;
    const int64_t t = (block << (8 - a.log_cols)) + (threadIdx.x >> a.log_cols);
    const int c = V * ((int)(blockIdx.x - block * a.chunks) * 256 + (int)(threadIdx.x & (a.cols - 1)));
    if (t >= a.tokens || c >= a.dim) return;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    for (int k = 0; k < a.top; ++k) {
        const int s = a.slot[t * a.top + k];
        if ((unsigned)s >= (unsigned)a.rows) continue;
        const float w = a.weights ? a.weights[t * a.top + k] : 1.0f;
        const float *y = a.y + s * a.ldy + c;
        float v[V];
        if constexpr (V == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(y);
        else v[0] = y[0];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(w, v[i], acc[i]);
    }
    if (a.add) {
        const float *y = a.add + t * a.lda + c;
        float v[V];
        if constexpr (V == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(y);
        else v[0] = y[0];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += v[i];
    }
    struct alignas(V * sizeof(T)) Out { T v[V]; } o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = from_f32<T>(acc[i]);
    *reinterpret_cast<Out *>(static_cast<T *>(a.out) + t * a.ldo + c) = o;
}

// ---- launches ----

template <typename KEY, int LPT, int VPL>
int launch_route_as(const RouteArgs &a, hipStream_t st)
{
    const size_t each = a.groups > 1 ? (size_t)(a.experts + a.groups) * sizeof(KEY) : 0;
    const int threads = each * (256 / LPT) > 65536 ? 64 : 256, per = threads / LPT;
    route_kernel<KEY, LPT, VPL><<<(unsigned)eif_ceil_div(a.tokens, per), threads, each * per, st>>>(a);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

template <typename KEY>
int launch_route(const RouteArgs &a, hipStream_t st)
{
    if (a.experts <= 256 && a.top <= 16 && a.tokens >= 1024) {
        if (a.experts <= 32) return launch_route_as<KEY, 16, 2>(a, st);
        if (a.experts <= 64) return launch_route_as<KEY, 16, 4>(a, st);
        if (a.experts <= 128) return launch_route_as<KEY, 16, 8>(a, st);
        return launch_route_as<KEY, 16, 16>(a, st);
    }
    if (a.experts <= 64) return launch_route_as<KEY, 64, 1>(a, st);
    if (a.experts <= 128) return launch_route_as<KEY, 64, 2>(a, st);
    if (a.experts <= 256) return launch_route_as<KEY, 64, 4>(a, st);
    if (a.experts <= 512) return launch_route_as<KEY, 64, 8>(a, st);
    if (a.experts <= 1024) return launch_route_as<KEY, 64, 16>(a, st);
    return launch_route_as<KEY, 64, 64>(a, st);
}

// Arguments of a sort; EIF_HIP_OK where it may be launched.
int check_sort(int tokens, int top, int experts, const int32_t *offsets, const int32_t *row, const int32_t *slot, const void *work,
               size_t work_bytes)
{
    if (tokens < 0 || top < 1 || experts < 1) return EIF_HIP_E_ARG;
    if (experts > kMaxExperts || top > kMaxExperts || (int64_t)tokens * top > kMaxPairs) return EIF_HIP_E_LIMIT;
    if (!offsets || !aligned(offsets, 4) || !aligned(row, 4) || !aligned(slot, 4) || !aligned(work, 4)) return EIF_HIP_E_ARG;
    if (tokens > 0 && (!row || !slot)) return EIF_HIP_E_ARG;
    const size_t need = eif_hip_moe_sort_bytes(tokens, top, experts);
    return need > 0 && (!work || work_bytes < need) ? EIF_HIP_E_ARG : EIF_HIP_OK;
}

int launch_sort(const int32_t *ids, int tokens, int top, int experts, int32_t *offsets, int32_t *row, int32_t *slot, void *work,
                hipStream_t st)
{
    const int pairs = tokens * top, blocks = sort_blocks(pairs), share = blocks > 1 ? sort_share(pairs) : pairs;
    int bits = 0;
    while (1 << bits < experts) ++bits;
    int32_t *counts = static_cast<int32_t *>(work);
    if (blocks > 1) {
        sort_count_kernel<<<blocks, 1024, experts * sizeof(int32_t), st>>>(ids, pairs, share, experts, counts);
        EIF_HIP_LAUNCHED();
    }
    const int waves = sort_waves(experts);
    const size_t lds = ((size_t)(waves + 1) * experts + 16) * sizeof(int32_t);
    sort_place_kernel<<<blocks, 64 * waves, lds, st>>>(ids, pairs, share, experts, bits, top, counts, blocks, offsets, row, slot);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

template <typename T>
int launch_combine(CombineArgs a, hipStream_t st)
{
    const bool vec = a.dim % 4 == 0 && aligned(a.y, 16) && a.ldy % 4 == 0 && (!a.add || (aligned(a.add, 16) && a.lda % 4 == 0)) &&
                     aligned(a.out, 4 * sizeof(T)) && a.ldo % 4 == 0;
    const int units = vec ? a.dim / 4 : a.dim;   // threads that a token's columns take
    a.log_cols = 0;
    while (a.log_cols < 8 && 1 << a.log_cols < units) ++a.log_cols;
    a.cols = 1 << a.log_cols;
    a.chunks = eif_ceil_div(units, 256);
    const int64_t blocks = ((int64_t)a.tokens + (256 >> a.log_cols) - 1) / (256 >> a.log_cols) * a.chunks;
    if (vec)
        combine_kernel<T, 4><<<(unsigned)blocks, 256, 0, st>>>(a);
    else
        combine_kernel<T, 1><<<(unsigned)blocks, 256, 0, st>>>(a);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

}  // namespace

extern "C" {

size_t eif_hip_moe_sort_bytes(int tokens, int top_k, int experts)
{
    if (tokens < 1 || top_k < 1 || experts < 1 || experts > kMaxExperts || top_k > kMaxExperts) return 0;
    const int64_t pairs = (int64_t)tokens * top_k;
    if (pairs > kMaxPairs) return 0;
    const int blocks = sort_blocks(pairs);
    return blocks > 1 ? (size_t)blocks * experts * sizeof(int32_t) : 0;
}

int eif_hip_moe_route(const void *logits, int type, int64_t ldl, int tokens, const eif_hip_moe_route_spec *spec, int32_t *ids,
                      float *weights, int32_t *offsets, int32_t *row, int32_t *slot, void *work, size_t work_bytes, void *stream)
{
    if (!spec || tokens < 0 || type < EIF_HIP_F32 || type > EIF_HIP_BF16) return EIF_HIP_E_ARG;
    const eif_hip_moe_route_spec s = *spec;
    if (s.experts < 1 || s.top_k < 1 || s.top_k > s.experts || ldl < s.experts) return EIF_HIP_E_ARG;
    if (s.score != EIF_HIP_SCORE_SOFTMAX && s.score != EIF_HIP_SCORE_SIGMOID) return EIF_HIP_E_ARG;
    if (s.groups < 1 || s.experts % s.groups != 0 || s.groups_kept < 1 || s.groups_kept > s.groups || s.group_best < 1 || s.group_best > 2)
        return EIF_HIP_E_ARG;
    if (!std::isfinite(s.scale) || !aligned(s.bias, 4)) return EIF_HIP_E_ARG;
    if (s.experts > kMaxExperts || s.top_k > kMaxTop || s.groups > kMaxGroups || tokens > kMaxTokens || (int64_t)tokens * s.top_k > kMaxPairs) return EIF_HIP_E_LIMIT;
    const bool sorted = offsets || row || slot;
    if (sorted) {
        const int rc = check_sort(tokens, s.top_k, s.experts, offsets, row, slot, work, work_bytes);
        if (rc) return rc;
    }
    if (tokens > 0 && (!logits || !ids || !weights)) return EIF_HIP_E_ARG;
    if (!aligned(logits, type == EIF_HIP_F32 ? 4 : 2) || !aligned(ids, 4) || !aligned(weights, 4)) return EIF_HIP_E_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (tokens > 0) {
        RouteArgs a{};
        a.logits = logits, a.bias = s.bias, a.ids = ids, a.weights = weights, a.ldl = ldl, a.type = type, a.tokens = tokens;
        a.experts = s.experts, a.top = s.top_k, a.score = s.score, a.renormalise = s.renormalise != 0, a.scale = s.scale;
        a.groups = s.groups_kept < s.groups ? s.groups : 1, a.kept = s.groups_kept, a.best = s.group_best;
        a.group_size = s.experts / s.groups;
        a.group_magic = (uint32_t)((0xffffffffull + a.group_size) / a.group_size);
        const bool wide = s.bias || (a.groups > 1 && a.best == 2);
        const int rc = wide ? launch_route<double>(a, st) : launch_route<float>(a, st);
        if (rc) return rc;
    }
    return sorted ? launch_sort(ids, tokens, s.top_k, s.experts, offsets, row, slot, work, st) : EIF_HIP_OK;
}

int eif_hip_moe_sort(const int32_t *ids, int tokens, int top_k, int experts, int32_t *offsets, int32_t *row, int32_t *slot, void *work,
                     size_t work_bytes, void *stream)
{
    const int rc = check_sort(tokens, top_k, experts, offsets, row, slot, work, work_bytes);
    if (rc) return rc;
    if ((tokens > 0 && !ids) || !aligned(ids, 4)) return EIF_HIP_E_ARG;
    return launch_sort(ids, tokens, top_k, experts, offsets, row, slot, work, (hipStream_t)stream);
}

int eif_hip_moe_combine(const float *y, int64_t ldy, int rows, const int32_t *slot, const float *weights, int tokens, int top_k,
                        const float *add, int64_t lda, int dim, void *out, int type, int64_t ldo, void *stream)
{
    if (tokens < 0 || rows < 0 || top_k < 1 || dim < 1 || type < EIF_HIP_F32 || type > EIF_HIP_BF16) return EIF_HIP_E_ARG;
    if (ldy < dim || ldo < dim || (add && lda < dim)) return EIF_HIP_E_ARG;
    if (dim > 1 << 24 || (int64_t)tokens * top_k > kMaxPairs || (int64_t)tokens * eif_ceil_div(dim, 256) > kLaunchBlocks)
        return EIF_HIP_E_LIMIT;
    if (tokens == 0) return EIF_HIP_OK;
    if ((rows > 0 && !y) || !slot || !out || !aligned(y, 4) || !aligned(slot, 4) || !aligned(weights, 4) || !aligned(add, 4) ||
        !aligned(out, type == EIF_HIP_F32 ? 4 : 2))
        return EIF_HIP_E_ARG;
    if (add == out && (type != EIF_HIP_F32 || lda != ldo)) return EIF_HIP_E_ARG;
    CombineArgs a{};
    a.y = y, a.weights = weights, a.add = add, a.slot = slot, a.out = out, a.ldy = ldy, a.lda = lda, a.ldo = ldo;
    a.rows = rows, a.tokens = tokens, a.top = top_k, a.dim = dim;
    hipStream_t st = (hipStream_t)stream;
    if (type == EIF_HIP_F32) return launch_combine<float>(a, st);
    return type == EIF_HIP_F16 ? launch_combine<__half>(a, st) : launch_combine<__hip_bfloat16>(a, st);
}

}  // extern "C"
