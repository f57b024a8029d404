// moe.hip -- routing to experts: the choice from a router's logits, pairs sorted by expert, the weighted sum of the experts' rows
// (eif_hip_moe.h).
#include "hip_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

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

// The value of lane l ^ LX.
template <int LX>
EIF_DEV uint32_t xlane_u(uint32_t v)
{
    if constexpr (LX <= 8) {
        return __float_as_uint(xlane<LX>(__uint_as_float(v)));
    } else {   // the swap of half waves, or of rows of 16, leaves both values in both halves
        const auto r = LX == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & LX) ? r[0] : r[1];
    }
}
template <int LX>
EIF_DEV float xlane_of(float v) { return __uint_as_float(xlane_u<LX>(__float_as_uint(v))); }
template <int LX>
EIF_DEV double xlane_of(double v)
{
    return __hiloint2double((int)xlane_u<LX>((uint32_t)__double2hiint(v)), (int)xlane_u<LX>((uint32_t)__double2loint(v)));
}
// The value of another lane of the row of 16, N lanes on around it.
template <int N>
EIF_DEV float row_turn(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false)); }
template <int N>
EIF_DEV double row_turn(double v)
{
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), 0x120 + N, 0xf, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), 0x120 + N, 0xf, 0xf, false));
}

// f of the integers FIRST .. LAST as types.
template <int FIRST, int LAST, typename F>
EIF_DEV void for_each(F f)
{
    if constexpr (FIRST <= LAST) {
        f(std::integral_constant<int, FIRST>{});
        for_each<FIRST + 1, LAST>(f);
    }
}

// f over the lanes l ^ 1, ^ 2, .. of a group of LPT lanes.
template <int LPT, typename F>
EIF_DEV void butterfly(F f)
{
    for_each<0, LPT == 64 ? 5 : 3>([&](auto i) { f(std::integral_constant<int, 1 << decltype(i)::value>{}); });
}
template <typename V>
EIF_DEV V larger(V a, V b) { return a > b ? a : b; }   // of numbers: nothing here is a NaN
template <int LPT, typename V>
EIF_DEV V lanes_max(V v)
{
    butterfly<LPT>([&](auto x) { v = larger(v, xlane_of<decltype(x)::value>(v)); });
    return v;
}
template <int LPT, typename V>
EIF_DEV V lanes_sum(V v)
{
    butterfly<LPT>([&](auto x) { v += xlane_of<decltype(x)::value>(v); });
    return v;
}

// e^x for x <= 709.7 to about an ulp: x = n ln 2 + r with ln 2 in two parts (Cody and Waite), e^r by its Taylor series up to r^13 / 13!,
// which |r| <= ln 2 / 2 leaves off by 5e-18. The library's function takes care of more and takes twice as long.
EIF_DEV double exp64(double x)
{
    x = larger(x, -760.0);   // 0 as well, and n fits
    const double n = rint(x * 1.4426950408889634);
    double r = fma(n, -0x1.62e42fefa3800p-1, x);   // 41 bits of ln 2, so that n times it is exact
    r = fma(n, -0x1.ef35793c76730p-45, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)n);
}

// 1 / d for 1 <= d < 2^1015: the instruction's 2^-26 or so and two Newton steps, each fused, so that the last rounds what it should.
EIF_DEV double reciprocal(double d)
{
    double q = __builtin_amdgcn_rcp(d);
    q = fma(fma(-d, q, 1.0), q, q);
    return fma(fma(-d, q, 1.0), q, q);
}

// 1 / (1 + e^-l): 0 from where e^-l leaves the range of 64 bits (l < -1024 ln 2), and e^l below -700, where the two are the same to
// 64 bits and the reciprocal comes near numbers that are not normal.
EIF_DEV double sigmoid64(double l)
{
    const bool far = l < -700.0;
    const double e = exp64(far ? l : -l), s = far ? e : reciprocal(1.0 + e);
    return l < -709.782712893384 ? 0.0 : s;
}

template <typename T>
EIF_DEV float logit_of(T v)
{
    const float l = (float)v;
    return l > -INFINITY ? fminf(l, 3.402823466e+38f) : -INFINITY;   // NaN and -inf: shut out
}
// Logits i LPT + sub of a row, i < VPL.
template <int LPT, int VPL, typename T>
EIF_DEV void load_logits(const T *row, int sub, int experts, float *l)
{
    T v[VPL];
    if (experts == LPT * VPL) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) v[i] = row[i * LPT + sub];
#pragma unroll
        for (int i = 0; i < VPL; ++i) l[i] = logit_of(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) v[i] = row[min(i * LPT + sub, experts - 1)];
#pragma unroll
        for (int i = 0; i < VPL; ++i) l[i] = i * LPT + sub < experts ? logit_of(v[i]) : -INFINITY;
    }
}

// What experts are compared by: their logits (no bias); score plus bias in 64 bits (experts of equal scores in 32 bits can differ in 64,
// and which of them is chosen changes the token's result by a whole expert); the same, sifted by sigmoids of 32 bits first.
enum { kByLogit, kByValue, kSifted };

// Candidates of a token that LDS holds: three a lane, or one.
constexpr int route_room(int lpt) { return lpt == 16 ? 48 : 64; }

// Bytes of LDS of a token: what the experts and groups are worth, later the candidates; and the lanes' largest. kSifted has the room of
// kByValue, which takes over where it cannot tell.
template <int MODE, int LPT>
__host__ __device__ constexpr int route_lds(int experts, int groups)
{
    const int room = route_room(LPT) * 16, worth = (experts + groups) * (MODE == kByLogit ? 4 : 8);
    return ((room > worth ? room : worth) + (LPT == 64 ? 64 * 8 : 0) + 15) / 16 * 16;
}

// Error of a sifting value: the sigmoid's is at most 1.9 2^-23 (exponent and sum rounded to 32 bits, the instructions' exponential and
// reciprocal an ulp off each), the sum's rounding 2^-24 of it.
EIF_DEV float sift_error(float v) { return fmaf(fabsf(v), 0x1.02p-24f, 0x1p-22f); }

// The groups whose experts may be chosen, a bit each, from what the experts are worth (val [experts], behind them room for the groups).
// SIFTED: `sure` says whether the kept ones are worth more than the others beyond any error. It is not known of a group whose sum leaves
// 32 bits, as that of two biases of the lowest value does.
template <int LPT, bool SIFTED, typename KEY>
EIF_DEV uint64_t kept_groups(const RouteArgs &a, int lane, KEY *val, bool &sure)
{
    const KEY none = -INFINITY;
    const int sub = lane % LPT;
    KEY *worth = val + a.experts;
    int share = 1;   // lanes that share a group: as many as there are for the power of two of groups
    while (share * 2 * a.groups <= LPT) share *= 2;
    wave_lds_order();
    for (int g0 = 0; g0 < a.groups; g0 += LPT) {
        const int g = g0 + sub / share, j = sub % share;
        KEY b1 = none, b2 = none;
        if (g < a.groups) {
            const KEY *of = val + g * a.group_size;
            int at = (j + g * share) % a.group_size;   // lanes start at different experts of their groups: different LDS banks
#pragma unroll 4
            for (int k = j; k < a.group_size; k += share) {
                const KEY v = of[at];
                at += share;
                if (at >= a.group_size) at -= a.group_size;
                const bool first = v > b1;
                b2 = first ? b1 : larger(b2, v);
                b1 = first ? v : b1;
            }
        }
        butterfly<LPT>([&](auto x) {
            if (decltype(x)::value < share) {
                const KEY o1 = xlane_of<decltype(x)::value>(b1), o2 = xlane_of<decltype(x)::value>(b2);
                b2 = larger(o1 > b1 ? b1 : o1, larger(b2, o2));
                b1 = larger(b1, o1);
            }
        });
        if (g < a.groups && j == 0) {
            const bool both = a.best == 2 && b2 > none;
            worth[g] = both ? b1 + b2 : b1;
            if constexpr (SIFTED) {   // of a group that is shut out: none
                const float off = sift_error(b1) + (both ? sift_error(b2) + fabsf(b1 + b2) * 0x1.02p-24f : 0.0f);
                worth[a.groups + g] = b1 > none ? off : 0.0f;
            }
        }
    }
    wave_lds_order();
    uint64_t keep = 0;
    KEY kept_least = INFINITY, dropped_most = none;
    bool known = true;
    for (int g0 = 0; g0 < a.groups; g0 += LPT) {
        const int g = g0 + sub;
        int better = a.kept;
        if (g < a.groups) {
            const KEY w = worth[g];
            better = 0;
#pragma unroll 4
            for (int h = 0; h < a.groups; ++h) better += worth[h] > w || (worth[h] == w && h < g);
            if constexpr (SIFTED) {
                const float off = worth[a.groups + g];   // finite only where what it is worth is, and 0 of a group that is shut out
                known = known && off < INFINITY;
                if (better < a.kept) kept_least = fminf(kept_least, w - off);
                else dropped_most = larger(dropped_most, w + off);
            }
        }
        const uint64_t bits = __ballot(better < a.kept);
        keep |= LPT == 64 ? bits : ((bits >> (lane & 48)) & 0xffff) << g0;
    }
    if constexpr (SIFTED) {
        const float least = -lanes_max<LPT>(-kept_least), most = lanes_max<LPT>(dropped_most);
        sure = known && (least > most || !(most > none));
    }
    wave_lds_order();
    return keep;
}

EIF_DEV int group_of(const RouteArgs &a, uint32_t e) { return a.group_size == 1 ? e : __umulhi(e, a.group_magic); }

EIF_DEV float logit_at(const RouteArgs &a, int64_t i)
{
    if (a.type == EIF_HIP_F32) return logit_of(static_cast<const float *>(a.logits)[i]);
    return a.type == EIF_HIP_F16 ? logit_of(static_cast<const __half *>(a.logits)[i]) : logit_of(static_cast<const __hip_bfloat16 *>(a.logits)[i]);
}

// What an expert is worth in 64 bits: its score, plus the bias; -inf where it is shut out. md, inverse: softmax.
EIF_DEV double value_of(const RouteArgs &a, float l, int e, double md, double inverse)
{
    const double s = a.score == EIF_HIP_SCORE_SOFTMAX ? (l > -INFINITY ? exp64((double)l - md) * inverse : 0.0) : sigmoid64(l);
    const double b = a.bias ? (double)a.bias[e] : 0.0;
    return l > -INFINITY && b > -INFINITY ? s + b : -INFINITY;
}

// The choice of any number of experts and of any equals: they stay in LDS, and the largest is taken top times over. Lane k gets the k-th.
template <int LPT, typename KEY>
EIF_DEV void choose_plainly(const RouteArgs &a, int64_t row, int lane, KEY *val, double md, double inverse, int &chosen, float &logit)
{
    constexpr bool by_value = sizeof(KEY) == 8;
    const KEY none = -INFINITY;
    const int sub = lane % LPT;
    wave_lds_order();
#pragma unroll 4
    for (int e = sub; e < a.experts; e += LPT) {
        const float l = logit_at(a, row + e);
        if constexpr (by_value) val[e] = value_of(a, l, e, md, inverse);
        else val[e] = l;
    }
    if (a.groups > 1 || (by_value && !a.bias)) {
        bool sure;
        const uint64_t keep = a.groups > 1 ? kept_groups<LPT, false>(a, lane, val, sure) : ~0ull;
#pragma unroll 1
        for (int e = sub; e < a.experts; e += LPT) {
            if (!((keep >> (a.groups > 1 ? group_of(a, e) : 0)) & 1)) val[e] = none;
            else if (by_value && !a.bias) val[e] = logit_at(a, row + e);   // the groups alone go by the scores
        }
    }
    chosen = -1;
#pragma unroll 1
    for (int k = 0; k < a.top; ++k) {
        wave_lds_order();
        KEY best = none;
        int at = INT32_MAX;
#pragma unroll 4
        for (int e = sub; e < a.experts; e += LPT) {
            const KEY v = val[e];
            at = v > best ? e : at;
            best = larger(best, v);
        }
        butterfly<LPT>([&](auto x) {
            constexpr int X = decltype(x)::value;
            const KEY ob = xlane_of<X>(best);
            const int oe = (int)xlane_u<X>((uint32_t)at);
            if (ob > best || (ob == best && oe < at)) {
                best = ob;
                at = oe;
            }
        });
        if (at == INT32_MAX) continue;
        if (sub == k) chosen = at;
        if (at % LPT == sub) val[at] = none;
    }
    if (chosen >= 0) logit = logit_at(a, row + chosen);
}

// LPT lanes a token, lane `sub` of them has experts sub, sub + LPT, .. (VPL of them; 0: any number, chosen plainly).
//   The choice: the top-th largest of the lanes' largest is at most the top-th largest of all, so that the experts at or above it hold the
// chosen ones, and are few more. They go to LDS, and each counts those that come before it. Sifted: the candidates are those within
// the error of 32 bits, and only they are computed in 64, an expert a lane in place of all, or the groups where two of them are nearer to
// each other than that error. Candidates beyond the room in LDS are chosen plainly: many equals; of 256 experts, a third of the waves
// where 16 lanes choose 15, and nine in ten where they choose 16 (some 48 candidates a token); most tokens where 64 lanes choose more than 44.
//   Bound by the vector instructions, 1300 a wave of four tokens and 256 experts with a bias and groups: 16001 tokens 15 us, 18 where two
// groups of some token have to be told apart in 64 bits (22 with all experts in 64 bits), 12.6 without groups, 9.8 by logits (15.4 where a
// softmax over all is not renormalised and each exponential is of 64 bits), where reading them takes 3.3. A few tokens are one wave's
// chain: 64 tokens 6.1 us.
template <int MODE, int LPT, int VPL>
EIF_DEV void route_token(const RouteArgs &a, int64_t token, bool live, int lane, char *lds)
{
    typedef typename std::conditional<MODE == kByValue, double, float>::type KEY;
    typedef typename std::conditional<MODE == kByLogit, float, double>::type VALUE;   // of a candidate
    constexpr int kRoom = route_room(LPT), kEach = VPL > 0 ? VPL : 1;
    const KEY none = -INFINITY;
    const int sub = lane % LPT;
    const int64_t row = token * a.ldl;

    int chosen = -1;   // lane k: the token's k-th expert, and its logit
    float logit = -INFINITY;
    bool plainly = VPL == 0;
    double md = 0.0, zd = 1.0;   // softmax: largest logit, sum of e^(l - m)
    const bool over_all = a.score == EIF_HIP_SCORE_SOFTMAX && (MODE == kByValue || !a.renormalise);
    if constexpr (VPL == 0) {
        if (over_all) {
            float m = -INFINITY;
#pragma unroll 4
            for (int e = sub; e < a.experts; e += LPT) m = larger(m, logit_at(a, row + e));
            m = lanes_max<LPT>(m);
            md = m == -INFINITY ? 0.0f : m;
            zd = 0.0;
#pragma unroll 2
            for (int e = sub; e < a.experts; e += LPT) {
                const float l = logit_at(a, row + e);
                zd += l > -INFINITY ? exp64((double)l - md) : 0.0;
            }
            zd = lanes_sum<LPT>(zd);
        }
    } else {
        float l[kEach];
        KEY by[kEach];
        if (a.type == EIF_HIP_F32) load_logits<LPT, kEach>(static_cast<const float *>(a.logits) + row, sub, a.experts, l);
        else if (a.type == EIF_HIP_F16) load_logits<LPT, kEach>(static_cast<const __half *>(a.logits) + row, sub, a.experts, l);
        else load_logits<LPT, kEach>(static_cast<const __hip_bfloat16 *>(a.logits) + row, sub, a.experts, l);
        if (over_all) {
            float m = l[0];
#pragma unroll
            for (int i = 1; i < VPL; ++i) m = larger(m, l[i]);
            m = lanes_max<LPT>(m);
            md = m == -INFINITY ? 0.0f : m;
        }
        KEY *val = reinterpret_cast<KEY *>(lds);
        if constexpr (MODE == kByValue) {
            double p[kEach];
            if (a.score == EIF_HIP_SCORE_SOFTMAX) {
                zd = 0.0;
#pragma unroll
                for (int i = 0; i < VPL; ++i) {
                    p[i] = l[i] > -INFINITY ? exp64((double)l[i] - md) : 0.0;
                    zd += p[i];
                }
                zd = lanes_sum<LPT>(zd);
                const double inverse = 1.0 / zd;
#pragma unroll
                for (int i = 0; i < VPL; ++i) p[i] *= inverse;
            } else {
#pragma unroll
                for (int i = 0; i < VPL; ++i) p[i] = sigmoid64(l[i]);
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = i * LPT + sub;
                const double b = a.bias && e < a.experts ? (double)a.bias[e] : 0.0;
                const bool open = l[i] > -INFINITY && b > -INFINITY;
                p[i] = open ? p[i] + b : none;
                by[i] = !open ? none : a.bias ? p[i] : (double)l[i];
                if (a.groups > 1 && e < a.experts) val[e] = p[i];
            }
        } else if constexpr (MODE == kSifted) {
            float b[kEach];
#pragma unroll
            for (int i = 0; i < VPL; ++i) b[i] = a.bias[min(i * LPT + sub, a.experts - 1)];
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const int e = i * LPT + sub;
                const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[i] * -1.44269504f));
                const float v = fmaf(l[i], 0.0f, s + b[i]);   // a logit of -inf makes it NaN
                by[i] = v > none ? v : none;
                if (a.groups > 1 && e < a.experts) val[e] = by[i];
            }
        } else {
            if (over_all) {
                zd = 0.0;
#pragma unroll
                for (int i = 0; i < VPL; ++i) zd += l[i] > -INFINITY ? exp64((double)l[i] - md) : 0.0;
                zd = lanes_sum<LPT>(zd);
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                by[i] = l[i];
                const int e = i * LPT + sub;
                if (a.groups > 1 && e < a.experts) val[e] = l[i];
            }
        }

        if (a.groups > 1) {
            bool sure = true;
            uint64_t keep = kept_groups<LPT, MODE == kSifted>(a, lane, val, sure);
            if constexpr (MODE == kSifted) {
                if (__ballot(!sure)) {   // 64 bits tell
                    double *value = reinterpret_cast<double *>(lds);
                    float b[kEach];
#pragma unroll
                    for (int i = 0; i < VPL; ++i) b[i] = a.bias[min(i * LPT + sub, a.experts - 1)];
#pragma unroll
                    for (int i = 0; i < VPL; ++i) {
                        const int e = i * LPT + sub;
                        const double v = sigmoid64(l[i]) + (double)b[i];
                        if (e < a.experts) value[e] = l[i] > -INFINITY && b[i] > none ? v : -INFINITY;
                        __builtin_amdgcn_sched_barrier(0);   // one after the other, for the registers' sake
                    }
                    keep = kept_groups<LPT, false>(a, lane, value, sure);
                }
            }
            if (a.group_size % LPT == 0) {   // a lane's i-th expert is of the same group in every lane
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (!((keep >> (i * LPT / a.group_size & 63)) & 1)) by[i] = none;
            } else {
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (!((keep >> (group_of(a, i * LPT + sub) & 63)) & 1)) by[i] = none;
            }
        }

        VALUE *at_value = reinterpret_cast<VALUE *>(lds);
        int *at_expert = reinterpret_cast<int *>(lds + kRoom * 8);
        float *at_logit = reinterpret_cast<float *>(at_expert + kRoom);
        KEY floor = by[0];
#pragma unroll
        for (int i = 1; i < VPL; ++i) floor = larger(floor, by[i]);
        {
            const KEY v = floor;
            int above = 0;   // lanes with a larger one
            if constexpr (LPT == 16) {
                for_each<1, 15>([&](auto n) { above += row_turn<decltype(n)::value>(v) > v; });
            } else {
                KEY *top = reinterpret_cast<KEY *>(lds + route_lds<MODE, LPT>(a.experts, a.groups) - 64 * 8);
                top[sub] = v;
                wave_lds_order();
#pragma unroll 16
                for (int j = 0; j < 64; ++j) above += top[j] > v;
            }
            floor = above < a.top ? v : (KEY)INFINITY;
            butterfly<LPT>([&](auto x) {
                const KEY o = xlane_of<decltype(x)::value>(floor);
                floor = o < floor ? o : floor;
            });
            if constexpr (MODE == kSifted) floor = floor < INFINITY ? floor - 2.0f * sift_error(floor) : floor;
        }
        int n = 0;   // candidates, in the order of their experts
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const bool in = by[i] >= floor && by[i] > none;
            const uint64_t all = __ballot(in);
            const uint32_t lo = LPT == 64 ? (uint32_t)all : (uint32_t)(all >> (lane & 48)) & 0xffff, hi = LPT == 64 ? (uint32_t)(all >> 32) : 0;
            const int before = LPT == 64 ? __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, n)) : n + __popc(lo & ((1u << sub) - 1));
            if (in && before < kRoom) {
                if constexpr (MODE != kSifted) at_value[before] = by[i];
                at_expert[before] = i * LPT + sub;
                at_logit[before] = l[i];
            }
            n += __popc(lo) + __popc(hi);
        }
        wave_lds_order();
        plainly = plainly || __ballot(n > kRoom) != 0;
        if (!plainly) {
            // the candidates that come before each of a lane's, and the chosen ones to their places
            constexpr int C = kRoom / LPT;
            int e[C], place[C];
            float le[C];
            VALUE v[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int k = sub + c * LPT;
                place[c] = a.top;
                if (k < n) {
                    e[c] = at_expert[k], le[c] = at_logit[k];
                    if constexpr (MODE == kSifted) at_value[k] = v[c] = sigmoid64(le[c]) + (double)a.bias[e[c]];
                    else v[c] = at_value[k];
                }
            }
            wave_lds_order();
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int k = sub + c * LPT;
                if (k < n) {
                    int before = 0;
#pragma unroll 4
                    for (int j = 0; j < n; ++j) {
                        const VALUE o = at_value[j];
                        before += o > v[c] || (o == v[c] && j < k);
                    }
                    place[c] = before;
                }
            }
            wave_lds_order();
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (place[c] < a.top) at_expert[place[c]] = e[c], at_logit[place[c]] = le[c];
            wave_lds_order();
            if (sub < min(a.top, n)) chosen = at_expert[sub], logit = at_logit[sub];
        }
    }
    if (plainly) choose_plainly<LPT>(a, row, lane, reinterpret_cast<VALUE *>(lds), md, 1.0 / zd, chosen, logit);

    // the weights, a lane each, in 64 bits
    const bool there = chosen >= 0;
    double w = 0.0;
    if (a.score == EIF_HIP_SCORE_SOFTMAX) {
        if (a.renormalise) md = lanes_max<LPT>(there ? logit : -INFINITY);
        w = there ? exp64((double)logit - md) : 0.0;
        if (a.renormalise) zd = lanes_sum<LPT>(w);
    } else {
        w = there ? sigmoid64(logit) : 0.0;
        zd = a.renormalise ? lanes_sum<LPT>(w) : 1.0;
    }
    if (live && sub < a.top) {
        a.ids[token * a.top + sub] = chosen;
        a.weights[token * a.top + sub] = w > 0.0 ? (float)(w / zd * (double)a.scale) : 0.0f;
    }
}

template <int MODE, int LPT, int VPL>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a)
{
    extern __shared__ char route_bytes[];
    const int mine = threadIdx.x / LPT;   // of the workgroup's tokens
    const int64_t token = (int64_t)blockIdx.x * (blockDim.x / LPT) + mine;
    route_token<MODE, LPT, VPL>(a, token < a.tokens ? token : a.tokens - 1, token < a.tokens, threadIdx.x & 63,
                                route_bytes + mine * route_lds<MODE, LPT>(a.experts, a.groups));
}

// ---- pairs by expert ----

constexpr int kSortBlocks = 256;      // of a sort in two launches, at most: one a CU
// Pairs that one workgroup sorts in one launch: a thousand more take it a microsecond (4000 of 64 experts 6.3 us, 8000 of 128 10.6), two
// launches take 6.6 and 8.3 us there.
constexpr int kSortAlone = 4096;
constexpr int kHeld = 4;              // of a wave's runs of 64 pairs, in registers

// Waves of a placing workgroup: one for 64 pairs, up to 16 with a counter of every expert in LDS each, 64 KB in all.
int sort_waves(int experts, int pairs)
{
    int waves = experts > 2048 ? 2 : experts > 1024 ? 4 : experts > 512 ? 8 : 16;
    while (waves > 1 && (waves / 2) * 64 >= pairs) waves /= 2;
    return waves;
}
// Pairs of a workgroup, whole steps of its waves: 1024, more from 128 workgroups on, whose counts each of them adds up (us of both
// launches with 1024 / 2048 / 4096: 16384 pairs of 64 experts 8.0 / 9.0 / -; 65536 of 256 9.5 / 9.8 / 12.4; 262144 of 128 11.4 / 10.7 /
// 11.7).
int sort_share(int64_t pairs)
{
    int64_t per = std::min<int64_t>((pairs + 127) / 128, 4096);
    per = std::max<int64_t>({per, 1024, (pairs + kSortBlocks - 1) / kSortBlocks});
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
// 262144 pairs of 128 experts 8.0 us behind 2.4 of counting, 66 of 8 2.8 us alone: a chain of barriers, loads and LDS, not of bytes.
// cnt: [waves][experts], then the sums [experts], those of workgroups before [experts], and of the waves [16].
EIF_DEV void sort_place(const int32_t *ids, int pairs, int share, int experts, int bits, int top, const int32_t *counts, int blocks,
                        int32_t *offsets, int32_t *row, int32_t *slot, int32_t *cnt)
{
    const int threads = blockDim.x, waves = threads >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int32_t *sums = cnt + waves * experts, *before = sums + experts, *part = before + experts;
    int32_t *own = cnt + wave * experts;
    const int lo = blockIdx.x * share, n = min(pairs - lo, share), run = (n + waves * 64 - 1) / (waves * 64) * 64;
    const int from = min(wave * run, n), to = min(from + run, n);
    int held[kHeld];   // the wave's first pairs stay in registers
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const int i = from + h * 64 + lane;
        held[h] = i < to ? ids[lo + i] : -1;
    }
    for (int i = threadIdx.x; i < (waves + 2) * experts; i += threads) cnt[i] = 0;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
        if ((unsigned)held[h] < (unsigned)experts) atomicAdd(&own[held[h]], 1);
    for (int i = from + kHeld * 64 + lane; i < to; i += 64) {
        const int id = ids[lo + i];
        if ((unsigned)id < (unsigned)experts) atomicAdd(&own[id], 1);
    }
    if (blocks > 1) {
        // the other workgroups' counts: all threads at once, eight loads of each under way (one thread an expert, a load after the
        // other, took 12 of 21 us with 64 workgroups and 128 experts)
        const int parts = max(1, threads / experts), per = (blocks + parts - 1) / parts;
        for (int i = threadIdx.x; i < parts * experts; i += threads) {
            const int p = i / experts, e = i - p * experts, b1 = min((p + 1) * per, blocks);
            int first = 0, all = 0;
#pragma unroll 8
            for (int b = p * per; b < b1; ++b) {
                const int c = counts[b * experts + e];
                first += b < (int)blockIdx.x ? c : 0;
                all += c;
            }
            atomicAdd(&before[e], first);
            atomicAdd(&sums[e], all);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += threads) {
        int at = before[e], c[16];
#pragma unroll
        for (int w = 0; w < 16; ++w) c[w] = w < waves ? cnt[w * experts + e] : 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < waves) cnt[w * experts + e] = at;
            at += c[w];
        }
        if (blocks == 1) sums[e] = at;
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
    const auto place = [&](int i, int id) {
        const int p = lo + i + lane;
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
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
        if (from + h * 64 < to) place(from + h * 64, held[h]);
    for (int i = from + kHeld * 64; i < to; i += 64) place(i, i + lane < to ? ids[lo + i + lane] : -1);
}

__global__ __launch_bounds__(1024) void sort_place_kernel(const int32_t *ids, int pairs, int share, int experts, int bits, int top,
                                                          const int32_t *counts, int blocks, int32_t *offsets, int32_t *row, int32_t *slot)
{
    extern __shared__ int32_t sort_words[];
    sort_place(ids, pairs, share, experts, bits, top, counts, blocks, offsets, row, slot, sort_words);
}

// A few tokens: one workgroup chooses for all of them at once and sorts what it chose, one launch in place of two: one token of 32
// experts 4.7 us in place of 2.5 and 2.8, 64 of 64 7.3 in place of 4.3 and 4.0.
template <int MODE, int LPT, int VPL>
__global__ __launch_bounds__(1024) void route_sort_kernel(RouteArgs a, int bits, int32_t *offsets, int32_t *row, int32_t *slot)
{
    extern __shared__ char route_bytes[];
    const int64_t token = threadIdx.x / LPT;
    route_token<MODE, LPT, VPL>(a, token < a.tokens ? token : a.tokens - 1, token < a.tokens, threadIdx.x & 63,
                                route_bytes + token * route_lds<MODE, LPT>(a.experts, a.groups));
    __syncthreads();   // the ids are in memory for the workgroup's other waves
    const int pairs = a.tokens * a.top;
    sort_place(a.ids, pairs, pairs, a.experts, bits, a.top, nullptr, 1, offsets, row, slot, reinterpret_cast<int32_t *>(route_bytes));
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

// A thread has four adjacent columns of a token (of the row's last ones fewer), 16 bytes at a time: rows that are not ALIGNED to them
// too, which loads of 16 bytes at any float and stores at any element serve (2000 tokens of 8 rows of 2047 32.7 us, with a
// column a thread 45.7). Bound by memory: 2048 tokens of 8 rows of 2048 with a residual, to bf16, 31.4 us, 5.0 TB/s of what it reads
// and writes, which is what a large copy reaches (34 us a row after the other in place of four at a time; a few tokens 3.1 in place of
// 3.5).
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a)
{
    struct alignas(ALIGNED ? 16 : 4) In { float v[4]; };
    struct alignas(ALIGNED ? 4 * sizeof(T) : sizeof(T)) Out { T v[4]; };
    const int64_t block = blockIdx.x / a.chunks;
    const int64_t t = (block << (8 - a.log_cols)) + (threadIdx.x >> a.log_cols);
    const int c = 4 * ((int)(blockIdx.x - block * a.chunks) * 256 + (int)(threadIdx.x & (a.cols - 1)));
    if (t >= a.tokens || c >= a.dim) return;
    const int n = ALIGNED ? 4 : min(a.dim - c, 4);
    const auto load = [&](const float *y) {
        if (n == 4) return *reinterpret_cast<const In *>(y);
        In r{};
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) r.v[i] = y[i];
        return r;
    };
    float acc[4] = {};
    const int32_t *slot = a.slot + t * a.top;
    for (int k0 = 0; k0 < a.top; k0 += 4) {   // four rows under way
        int s[4];
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = min(k0 + k, a.top - 1);
            s[k] = slot[at];
            w[k] = a.weights ? a.weights[t * a.top + at] : 1.0f;
            if (k0 + k >= a.top) s[k] = -1;
        }
        In v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if ((unsigned)s[k] < (unsigned)a.rows) v[k] = load(a.y + s[k] * a.ldy + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if ((unsigned)s[k] < (unsigned)a.rows) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = fmaf(w[k], v[k].v[i], acc[i]);
            }
        }
    }
    if (a.add) {
        const In v = load(a.add + t * a.lda + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += v.v[i];
    }
    Out o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = from_f32<T>(acc[i]);
    T *out = static_cast<T *>(a.out) + t * a.ldo + c;
    if (n == 4) {
        *reinterpret_cast<Out *>(out) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) out[i] = o.v[i];
    }
}

// ---- launches ----

int bits_of(int experts)
{
    int bits = 0;
    while (1 << bits < experts) ++bits;
    return bits;
}

// LDS of a placing workgroup.
size_t sort_lds(int waves, int experts) { return ((size_t)(waves + 2) * experts + 16) * sizeof(int32_t); }

// Where the sorted pairs of a choice go; offsets NULL: nowhere.
struct SortedTo {
    int32_t *offsets, *row, *slot;
    void *work;
};

int launch_sort(const int32_t *ids, int tokens, int top, int experts, const SortedTo &to, hipStream_t st)
{
    const int pairs = tokens * top, blocks = sort_blocks(pairs), share = blocks > 1 ? sort_share(pairs) : pairs;
    int32_t *counts = static_cast<int32_t *>(to.work);
    if (blocks > 1) {
        sort_count_kernel<<<blocks, 1024, experts * sizeof(int32_t), st>>>(ids, pairs, share, experts, counts);
        EIF_HIP_LAUNCHED();
    }
    const int waves = sort_waves(experts, share);
    sort_place_kernel<<<blocks, 64 * waves, sort_lds(waves, experts), st>>>(ids, pairs, share, experts, bits_of(experts), top, counts, blocks,
                                                                            to.offsets, to.row, to.slot);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

template <int MODE, int LPT, int VPL>
int launch_route_as(const RouteArgs &a, const SortedTo &to, hipStream_t st)
{
    const size_t each = route_lds<MODE, LPT>(a.experts, a.groups);
    if constexpr (VPL > 0) {
        // one launch with the sort where one workgroup's waves have room for every token and its counters; not with 16 waves of 64 lanes
        // a token, whose time on one CU passes that of two launches (16 tokens of 256 experts 11.0 us, 6.1 and 3.5 on many)
        const int waves = eif_ceil_div(a.tokens, 64 / LPT);
        const size_t lds = std::max(each * std::min(waves, 16) * (64 / LPT), sort_lds(std::min(waves, 16), a.experts));
        if (to.offsets && waves <= (LPT == 16 ? 16 : 8) && lds <= 65536) {
            route_sort_kernel<MODE, LPT, VPL><<<1, 64 * waves, lds, st>>>(a, bits_of(a.experts), to.offsets, to.row, to.slot);
            EIF_HIP_LAUNCHED();
            return EIF_HIP_OK;
        }
    }
    // one wave a workgroup where there are few, so that they spread over the CUs, and where LDS would not hold four
    const int threads = a.tokens <= 4096 || each * (256 / LPT) > 65536 ? 64 : 256, per = threads / LPT;
    route_kernel<MODE, LPT, VPL><<<(unsigned)eif_ceil_div(a.tokens, per), threads, each * per, st>>>(a);
    EIF_HIP_LAUNCHED();
    return to.offsets ? launch_sort(a.ids, a.tokens, a.top, a.experts, to, st) : EIF_HIP_OK;
}

// Lanes of a token: 16, so that its fixed work is shared by four tokens of a wave, or 64 where there are few tokens, whose time is one
// wave's (us, 16 / 64: 64 tokens of 256 experts with a bias and groups 8.9 / 6.5, without 6.9 / 4.8; 2000 9.0 / 7.2, 4000 9.3 / 9.7;
// one token of 32 3.0 / 3.5). Those are of 8 experts a token. Of 16 the candidates pass the room of 16 lanes: 16001 tokens of 256 experts by
// logits 10.8 us for 8, 17.6 for 13, 27.6 for 16, and 14.9 for 17 on 64 lanes; sifted 12.6, 24, 40 and 17.5. 64 of 512 experts take 203 and
// 281 us, chosen plainly.
template <int MODE>
int launch_route(const RouteArgs &a, const SortedTo &to, hipStream_t st)
{
    if (a.experts <= (a.tokens <= 2048 ? 64 : 256) && a.top <= 16) {
        if (a.experts <= 32) return launch_route_as<MODE, 16, 2>(a, to, st);
        if (a.experts <= 64) return launch_route_as<MODE, 16, 4>(a, to, st);
        if (a.experts <= 128) return launch_route_as<MODE, 16, 8>(a, to, st);
        return launch_route_as<MODE, 16, 16>(a, to, st);
    }
    if (a.experts <= 256) return launch_route_as<MODE, 64, 4>(a, to, st);
    if (a.experts <= 512) return launch_route_as<MODE, 64, 8>(a, to, st);
    if (a.experts <= 1024) return launch_route_as<MODE, 64, 16>(a, to, st);
    return launch_route_as<MODE == kSifted ? kByValue : MODE, 64, 0>(a, to, st);
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

template <typename T>
int launch_combine(CombineArgs a, hipStream_t st)
{
    const bool whole = a.dim % 4 == 0 && aligned(a.y, 16) && a.ldy % 4 == 0 && (!a.add || (aligned(a.add, 16) && a.lda % 4 == 0)) &&
                     aligned(a.out, 4 * sizeof(T)) && a.ldo % 4 == 0;
    const int units = eif_ceil_div(a.dim, 4);   // threads that a token's columns take
    a.log_cols = 0;
    while (a.log_cols < 8 && 1 << a.log_cols < units) ++a.log_cols;
    a.cols = 1 << a.log_cols;
    a.chunks = eif_ceil_div(units, 256);
    const int64_t blocks = ((int64_t)a.tokens + (256 >> a.log_cols) - 1) / (256 >> a.log_cols) * a.chunks;
    if (whole)
        combine_kernel<T, true><<<(unsigned)blocks, 256, 0, st>>>(a);
    else
        combine_kernel<T, false><<<(unsigned)blocks, 256, 0, st>>>(a);
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
    const SortedTo to{offsets, row, slot, work};
    if (tokens > 0) {
        RouteArgs a{};
        a.logits = logits, a.bias = s.bias, a.ids = ids, a.weights = weights, a.ldl = ldl, a.type = type, a.tokens = tokens;
        a.experts = s.experts, a.top = s.top_k, a.score = s.score, a.renormalise = s.renormalise != 0, a.scale = s.scale;
        a.groups = s.groups_kept < s.groups ? s.groups : 1, a.kept = s.groups_kept, a.best = s.group_best;
        a.group_size = s.experts / s.groups;
        a.group_magic = (uint32_t)((0xffffffffull + a.group_size) / a.group_size);
        const bool by_value = s.bias || (a.groups > 1 && a.best == 2), sifted = s.bias && s.score == EIF_HIP_SCORE_SIGMOID;
        if (sifted) return launch_route<kSifted>(a, to, st);
        return by_value ? launch_route<kByValue>(a, to, st) : launch_route<kByLogit>(a, to, st);
    }
    return sorted ? launch_sort(ids, 0, s.top_k, s.experts, to, st) : EIF_HIP_OK;
}

int eif_hip_moe_sort(const int32_t *ids, int tokens, int top_k, int experts, int32_t *offsets, int32_t *row, int32_t *slot, void *work,
                     size_t work_bytes, void *stream)
{
    const int rc = check_sort(tokens, top_k, experts, offsets, row, slot, work, work_bytes);
    if (rc) return rc;
    if ((tokens > 0 && !ids) || !aligned(ids, 4)) return EIF_HIP_E_ARG;
    return launch_sort(ids, tokens, top_k, experts, SortedTo{offsets, row, slot, work}, (hipStream_t)stream);
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
