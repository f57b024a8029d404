// mx4.hip -- microscaled 4-bit (MXFP4) operators: quantisation of rows, resident matrices, products (eif_hip_mx.h).
#include "hip_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <new>
#include <type_traits>

#include "../../include/eif_hip_mx.h"

// A resident matrix: 16-row tiles, a tile's columns in spans of 256 (8 blocks of 32), two scaled MFMAs (16x16x128) each.
//   codes  [expert][tile][span][step 0..1][lane][16 bytes]: lane l has row l % 16, block 2 (l / 16) + step of the span, so
//          a wave's load is 1 KB in one run and its 16 bytes are the MFMA's operand. (Which column meets which MFMA does
//          not matter as long as both operands agree; this choice gives a lane of a row-major operand 32 consecutive
//          bytes of codes and two consecutive scale bytes a span.)
//   scales [expert][tile][pair of spans][lane][4 bytes]: the scale bytes of the lane's four blocks of the two spans.
// Rows beyond the matrix, columns beyond cols and the span that fills the last pair are zeros.
struct eif_hip_mx4_weight {
    uint8_t *codes;
    uint32_t *scales;
    int device, experts, rows, cols;
    int tiles, spans;   // of one matrix
    size_t bytes;
};

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kSpan = 256;

__host__ __device__ inline size_t tile_codes(int spans) { return (size_t)spans * 2048; }
__host__ __device__ inline size_t tile_scales(int spans) { return (size_t)((spans + 1) / 2) * 64; }   // dwords

// ---- quantisation ----

EIF_DEV uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The scale byte of a block from the bits of its largest magnitude (as integers, so that infinities and NaN win):
// max(0, E - 2) of its exponent field E, which is floor(log2 a) - 2 + 127 of a normal number; 255 where it is not finite.
EIF_DEV uint32_t scale_byte(uint32_t amax)
{
    const uint32_t e = amax >> 23;
    return e == 255 ? 255 : (e > 2 ? e - 2 : 0);
}

// 1 / 2^(b - 127), always a normal number (b <= 252); 0 for b = 255, whose codes are 0.
EIF_DEV float scale_inverse(uint32_t b) { return b == 255 ? 0.0f : __uint_as_float((254 - b) << 23); }

EIF_DEV float scale_value(uint32_t b) { return __uint_as_float(b == 255 ? 0x7fc00000u : b == 0 ? 0x00400000u : b << 23); }

// Four values times 1/scale -> four codes. v_cvt_scalef32_pk_fp4_f32 rounds to the nearest, ties to the even code, and
// saturates. A block that is not finite passes 0 as values.
EIF_DEV uint32_t codes4(const float *v, float inv, bool finite)
{
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = finite ? v[i] * inv : 0.0f;
    uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, t[0], t[1], 1.0f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, t[2], t[3], 1.0f, 1);
    return r;
}

EIF_DEV float to_f32(float v) { return v; }
EIF_DEV float to_f32(__half v) { return __half2float(v); }
EIF_DEV float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
struct alignas(4 * sizeof(T)) Quad { T v[4]; };

// Columns c .. c + 3 of a row, as they come (loads alone, so that several can be under way) ...
// VEC: x is aligned to four elements and cols a multiple of four. Columns behind the last are read within the row.
template <typename T, bool VEC>
EIF_DEV Quad<T> load4(const T *xr, int c, int cols)
{
    if constexpr (VEC) {
        return *reinterpret_cast<const Quad<T> *>(xr + (c < cols ? c : 0));
    } else {
        Quad<T> q;
#pragma unroll
        for (int i = 0; i < 4; ++i) q.v[i] = xr[min(c + i, cols - 1)];
        return q;
    }
}
// ... and as FP32, zeros behind the last.
template <typename T>
EIF_DEV void values4(const Quad<T> &q, int c, int cols, float *v)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i < cols ? to_f32(q.v[i]) : 0.0f;
}

// Four values of each lane, a block being eight lanes: the block's scale byte, and the lane's codes.
EIF_DEV uint32_t quantise4(const float *v, uint32_t &byte)
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = umax(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = umax(m, __float_as_uint(xlane<1>(__uint_as_float(m))));
    m = umax(m, __float_as_uint(xlane<2>(__uint_as_float(m))));
    m = umax(m, __float_as_uint(xlane<4>(__uint_as_float(m))));
    byte = scale_byte(m);
    return codes4(v, scale_inverse(byte), byte != 255);
}

// One wave a row and span: lane l has columns 4 l .. 4 l + 3, a block is eight lanes, and a wave's loads and stores are one run.
// Bound by memory: 3001x6912 FP32 with values 34.3 us, 5.2 TB/s of what it reads and writes (43 with values stored four bytes at
// a time); without values 20.6, 4.6 TB/s. Two to eight spans a wave, their loads first, were no faster (34.0 to 37.6) and small
// calls slower (64x2560 2.1 us with one, 2.5 with two). Not so 2-byte rows without values: 13824x2560 28.8 us (bf16) and 29.8 (f16),
// 3.0 TB/s, hardly less than the 34.0 of FP32 rows; there the waves' instructions count (all on inputs of more than 512 MB in turn).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T *x, int64_t ldx, int rows, int cols, int spans,
                                                         uint8_t *codes, int64_t ldc, uint8_t *scales, int64_t lds,
                                                         float *values, int64_t ldv, bool vec_values)
{
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), row = unit / spans;
    if (row >= rows) return;
    const int c = (int)(unit - row * spans) * kSpan + lane * 4;
    float v[4];
    values4(load4<T, VEC>(x + row * ldx, c, cols), c, cols, v);
    uint32_t b;
    const uint32_t q = quantise4(v, b);
    if (codes) {
        *reinterpret_cast<uint16_t *>(codes + row * ldc + (c >> 1)) = (uint16_t)q;
        if ((lane & 7) == 0) scales[row * lds + (c >> 5)] = (uint8_t)b;
    }
    if (values) {
        const float s = scale_value(b);
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
        const float o[4] = {lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
        float *vr = values + row * ldv + c;
        if (vec_values && c + 4 <= cols) {
            *reinterpret_cast<float4 *>(vr) = make_float4(o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < cols) vr[i] = o[i];
        }
    }
}

// ---- the resident layout ----

// One thread a 16-byte piece of the layout, from piece `first` on: its lane's row, block and step.
__global__ __launch_bounds__(256) void mx4_repack_kernel(const uint8_t *src, int64_t ldc, int rows, int cols, int tiles,
                                                         int spans, uint8_t *dst, size_t first, size_t pieces, bool vec)
{
    const size_t i = first + (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int lane = (int)(i & 63), step = (int)(i >> 6) & 1;
    size_t t = i >> 7;
    const int span = (int)(t % spans);
    t /= spans;
    const int row = (int)(t % tiles) * 16 + (lane & 15);
    const size_t e = t / tiles;
    const int c0 = span * kSpan + (2 * (lane >> 4) + step) * 32;
    uint32_t w[4] = {0, 0, 0, 0};
    if (row < rows) {
        const uint8_t *s = src + (int64_t)(e * rows + row) * ldc;
        if (vec && c0 + 32 <= cols) {   // rows aligned to 16 bytes
            reinterpret_cast<uint4 *>(dst)[i] = *reinterpret_cast<const uint4 *>(s + (c0 >> 1));
            return;
        }
        for (int j = 0; j < 16; ++j) {
            const int c = c0 + 2 * j;
            uint32_t v = c < cols ? s[c >> 1] : 0;
            if (c + 1 >= cols) v &= 0x0F;   // the last byte of an odd count holds one code
            w[j >> 2] |= v << (8 * (j & 3));
        }
    }
    reinterpret_cast<uint4 *>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

// One thread a dword of scales, from dword `first` on: the lane's four blocks of a pair of spans.
__global__ __launch_bounds__(256) void mx4_repack_scales_kernel(const uint8_t *src, int64_t lds, int rows, int cols,
                                                                int tiles, int spans, uint32_t *dst, size_t first, size_t n)
{
    const size_t i = first + (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int lane = (int)(i & 63), pairs = (spans + 1) / 2, blocks = (cols + 31) / 32;
    size_t t = i >> 6;
    const int pair = (int)(t % pairs);
    t /= pairs;
    const int row = (int)(t % tiles) * 16 + (lane & 15);
    const size_t e = t / tiles;
    uint32_t w = 0;
    for (int j = 0; j < 4; ++j) {
        const int block = (2 * pair + (j >> 1)) * 8 + 2 * (lane >> 4) + (j & 1);
        if (row < rows && block < blocks) w |= (uint32_t)src[(int64_t)(e * rows + row) * lds + block] << (8 * j);
    }
    dst[i] = w;
}

// ---- products ----

struct Mx4Args {
    const uint8_t *wc;
    const uint32_t *ws;
    int tiles, spans, rows;         // of one matrix; gated: rows and tiles of the stacked matrix
    const uint8_t *codes, *scales;  // operand rows
    int64_t ldc, lds;
    const float *bias;
    float *y;
    int64_t ldy;
    int M;
    int groups;                     // of token rows
    uint32_t code_bytes;            // of the operand rows' codes, 0 where they are 2^32 or more
    bool vec;                       // y takes 16-byte stores
    // by expert
    int experts, rows_in;
    const int32_t *index, *offsets;
    // rows form
    const void *x;
    int64_t ldx;
    int cols;
    bool vecx;                      // x takes loads of four elements
};

// One step of span H of a pair: a row tile's codes with their scale in byte 2 H + STEP of sw, operand rows' codes with
// theirs in byte STEP of sx.
template <int H, int STEP>
EIF_DEV v4f step_mfma(v4f acc, v4i w, uint32_t sw, v4i x, uint32_t sx)
{
    const v8i a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 2 * H + STEP, (int)sw, STEP, (int)sx);
}

template <int H>
EIF_DEV v4f span_mfma(v4f acc, v4i w0, v4i w1, uint32_t sw, v4i x0, v4i x1, uint32_t sx)
{
    return step_mfma<H, 1>(step_mfma<H, 0>(acc, w0, sw, x0, sx), w1, sw, x1, sx);
}

// SiLU(g) u. v_exp_f32 and v_rcp_f32 are within one unit in the last place; the roundings of log2(e) and of its product with g
// move the exponential by up to 2^-23 |g| of itself. Below g = -87.3 the reciprocal of 1 + e^-g is below the smallest normal number,
// which v_rcp_f32 gives as 0, and so is the output, where |SiLU(g)| is at most 87.4 2^-126. Forms without that end, with the whole
// part of the exponent applied last, cost 512 rows through gated 13824x2560 (15.0 us): without a branch 6 %, with one for each
// output 14 %, with one for a wave's tile 36 %; 16384 rows by expert through gated 2816x2048 (98 us) 4 to 6 %.
EIF_DEV float swiglu(float g, float u)
{
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * g);
    return (g * __builtin_amdgcn_rcpf(1.0f + e)) * u;
}

// The g-th group of TM token rows over the experts' ranges: its expert and its rows [lo, hi); false beyond the last.
// One wave's lanes take 64 experts at a time; a range is cut to [0, M], and a group taken only inside its range, so every
// row is in bounds whatever the offsets.
template <int TM>
EIF_DEV bool find_group(const Mx4Args &a, int g, int &expert, int &lo, int &hi)
{
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane;
        int s = 0, n = 0;
        if (e < a.experts) {
            s = min(max(a.offsets[e], 0), a.M);
            n = max(min(max(a.offsets[e + 1], 0), a.M) - s, 0);
        }
        const int groups = (n + TM - 1) / TM;
        int sum = groups;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(sum, d, 64);
            if (lane >= d) sum += v;
        }
        const unsigned long long past = __ballot(base + sum > g);
        if (past) {
            const int l = __ffsll(past) - 1;
            const int at = g - (base + __shfl(sum - groups, l, 64));
            const int s0 = __shfl(s, l, 64), n0 = __shfl(n, l, 64);
            if (at < 0 || at >= (n0 + TM - 1) / TM) return false;   // ranges that overlap, with sums beyond an int
            expert = __builtin_amdgcn_readfirstlane(e0 + l);
            lo = __builtin_amdgcn_readfirstlane(s0 + at * TM);
            hi = __builtin_amdgcn_readfirstlane(min(s0 + at * TM + TM, s0 + n0));
            return true;
        }
        base += __shfl(sum, 63, 64);
    }
    return false;
}

// The biases of a lane's four output rows r0 .. r0 + 3 (gated: gate's, then up's); rows behind the last get some bias.
template <bool GLU>
EIF_DEV void load_bias(const float *bias, int r0, int out_rows, float *b0, float *b1)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = min(r0 + j, out_rows - 1);
        b0[j] = bias[r];
        if (GLU) b1[j] = bias[out_rows + r];
    }
}

// The lane's four outputs of a token row.
template <bool GLU>
EIF_DEV void outputs(v4f s0, v4f s1, const float *b0, const float *b1, float *v)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = s0[j] + b0[j];
        if (GLU) v[j] = swiglu(v[j], s1[j] + b1[j]);
    }
}

// WHOLE: all four exist and y takes a 16-byte store.
template <bool GLU, bool WHOLE>
EIF_DEV void store_outputs(float *yr, int r0, int out_rows, v4f s0, v4f s1, const float *b0, const float *b1)
{
    float v[4];
    outputs<GLU>(s0, s1, b0, b1, v);
    if (WHOLE) {
        *reinterpret_cast<float4 *>(yr + r0) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (r0 + j < out_rows) yr[r0 + j] = v[j];
    }
}

// Few token rows: what counts is how soon and how much of the matrix is on its way. A workgroup of eight waves takes
// 8 / KW row tiles (gated: tiles of the gate's and the same of the up projection's) and 16 TT token rows. KW waves share a
// tile: wave k takes the spans k, k + KW, ..., D at a time with all their loads out at once, and the sums meet in LDS.
//   X void: quantised operand rows, straight from memory. Else the rows form: every workgroup quantises the (at most 8)
// rows of X into LDS while its first codes are on their way.
template <typename X, int TT, int KW, int D, bool GLU, bool GROUPED>
__global__ __launch_bounds__(512) void mx4_split_kernel(Mx4Args a)
{
    constexpr bool ROWS = !std::is_void<X>::value;
    constexpr int NT = GLU ? 2 : 1, TM = 16 * TT, TW = 8 / KW;
    __shared__ v4f red[KW == 1 ? 1 : 8][NT * TT][64];
    extern __shared__ __align__(16) uint8_t staged[];   // rows form: codes [M][spans 128 + 16], then scales [M][spans 8]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, slot = lane >> 4, kw = wave % KW;
    const int otiles = GLU ? a.tiles / 2 : a.tiles, tblocks = (otiles + TW - 1) / TW;
    const int group = blockIdx.x / tblocks, tile = (blockIdx.x % tblocks) * TW + wave / KW;
    int expert = 0, lo = group * TM, hi = min(lo + TM, a.M);
    if (GROUPED && !find_group<TM>(a, group, expert, lo, hi)) return;

    const uint8_t *wc[NT];
    const uint32_t *ws[NT];
#pragma unroll
    for (int h = 0; h < NT; ++h) {
        const size_t t = (size_t)expert * a.tiles + h * otiles + min(tile, otiles - 1);
        wc[h] = a.wc + t * tile_codes(a.spans);
        ws[h] = a.ws + t * tile_scales(a.spans);
    }
    struct Weights {
        v4i c[NT][2];
        uint32_t s[NT];
    };
    auto load_weights = [&](Weights &f, int p) {
#pragma unroll
        for (int h = 0; h < NT; ++h) {
            f.c[h][0] = *reinterpret_cast<const v4i *>(wc[h] + (size_t)p * 2048 + lane * 16);
            f.c[h][1] = *reinterpret_cast<const v4i *>(wc[h] + (size_t)p * 2048 + 1024 + lane * 16);
            f.s[h] = ws[h][(size_t)(p >> 1) * 64 + lane];
        }
    };
    // the j-th span of a wave's batch; behind the last one the batch's first again
    auto batch_span = [&](int p0, int j) { return p0 + j * KW < a.spans ? p0 + j * KW : min(p0, a.spans - 1); };
    Weights w[D];
#pragma unroll
    for (int j = 0; j < D; ++j) load_weights(w[j], batch_span(kw, j));
    __builtin_amdgcn_sched_barrier(0);   // the loads go out here

    const uint8_t *xr[TT];
    const uint8_t *sr[TT];
    bool ok[TT];
    if constexpr (ROWS) {
        const int ldq = a.spans * 128 + 16;   // 16 bytes on from row to row in the banks
        uint8_t *sc = staged + a.M * ldq;
        const X *x = static_cast<const X *>(a.x);
        auto stage = [&](auto vec) {
            constexpr int U = 4;   // rows and spans that a wave has under way
            for (int u0 = wave; u0 < a.M * a.spans; u0 += 8 * U) {
                Quad<X> q[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int u = min(u0 + 8 * i, a.M * a.spans - 1);
                    q[i] = load4<X, decltype(vec)::value>(x + u / a.spans * a.ldx, u % a.spans * kSpan + lane * 4, a.cols);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int u = u0 + 8 * i, row = u / a.spans, c = u % a.spans * kSpan + lane * 4;
                    if (u >= a.M * a.spans) break;
                    float v[4];
                    values4(q[i], c, a.cols, v);
                    uint32_t b;
                    const uint32_t code = quantise4(v, b);
                    *reinterpret_cast<uint16_t *>(staged + row * ldq + (c >> 1)) = (uint16_t)code;
                    if ((lane & 7) == 0) sc[row * a.spans * 8 + (c >> 5)] = (uint8_t)b;
                }
            }
        };
        if (a.vecx)
            stage(std::true_type{});
        else
            stage(std::false_type{});
        __syncthreads();
        ok[0] = n < a.M;
        const int row = ok[0] ? n : 0;
        xr[0] = staged + row * ldq + slot * 32;
        sr[0] = sc + row * a.spans * 8 + slot * 2;
    } else {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int m = lo + 16 * t + n;
            int r = m;
            ok[t] = m < hi;
            if (GROUPED) {
                if (ok[t] && a.index) r = a.index[m];
                ok[t] = ok[t] && r >= 0 && r < a.rows_in;
            }
            r = ok[t] ? r : 0;   // row 0 is there to be read; its sums are not stored
            xr[t] = a.codes + r * a.ldc + slot * 32;
            sr[t] = a.scales + r * a.lds + slot * 2;
        }
    }
    v4f acc[NT][TT] = {};
    for (int p0 = kw; p0 < a.spans; p0 += KW * D) {
        v4i x[D][TT][2];
        uint32_t sx[D][TT];
        if (p0 != kw) {
#pragma unroll
            for (int j = 0; j < D; ++j) load_weights(w[j], batch_span(p0, j));
        }
#pragma unroll
        for (int j = 0; j < D; ++j) {
            const int p = batch_span(p0, j);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                x[j][t][0] = *reinterpret_cast<const v4i *>(xr[t] + (size_t)p * 128);
                x[j][t][1] = *reinterpret_cast<const v4i *>(xr[t] + (size_t)p * 128 + 16);
                sx[j][t] = *reinterpret_cast<const uint16_t *>(sr[t] + (size_t)p * 8);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < D; ++j) {
            const int p = p0 + j * KW;
            if (p >= a.spans) break;
#pragma unroll
            for (int h = 0; h < NT; ++h)
#pragma unroll
                for (int t = 0; t < TT; ++t)
                    acc[h][t] = span_mfma<0>(acc[h][t], w[j].c[h][0], w[j].c[h][1], w[j].s[h] >> (16 * (p & 1)), x[j][t][0],
                                             x[j][t][1], sx[j][t]);
        }
    }
    if (KW > 1) {
#pragma unroll
        for (int h = 0; h < NT; ++h)
#pragma unroll
            for (int t = 0; t < TT; ++t) red[KW == 1 ? 0 : wave][h * TT + t][lane] = acc[h][t];
        __syncthreads();
    }
    if (tile >= otiles) return;
    const int out_rows = GLU ? a.rows / 2 : a.rows, r0 = tile * 16 + slot * 4;
    float b0[4] = {}, b1[4] = {};
    if (a.bias) load_bias<GLU>(a.bias + (size_t)expert * a.rows, r0, out_rows, b0, b1);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        if (KW > 1) {   // the waves of a tile take its token tiles in turn
            if (t % KW != kw) continue;
#pragma unroll
            for (int h = 0; h < NT; ++h) {
                acc[h][t] = red[wave - kw][h * TT + t][lane];
#pragma unroll
                for (int k = 1; k < KW; ++k) acc[h][t] += red[wave - kw + k][h * TT + t][lane];
            }
        }
        if (!ok[t]) continue;
        float *yr = a.y + (int64_t)(lo + 16 * t + n) * a.ldy;
        if (a.vec && r0 + 4 <= out_rows)
            store_outputs<GLU, true>(yr, r0, out_rows, acc[0][t], acc[NT - 1][t], b0, b1);
        else
            store_outputs<GLU, false>(yr, r0, out_rows, acc[0][t], acc[NT - 1][t], b0, b1);
    }
}

// Of 16 rows, two by two, the numbers 0 to 7 such that rows 0-3 and 12-15 have 0 to 3, rows 4-11 the others, and within
// each four a number's neighbour by exclusive-or 2.
__host__ __device__ constexpr int place(int row) { return (row & 6) ^ (row & 8 ? 5 : 0); }

// 16 bytes from memory straight into LDS, lane l's behind lane l - 1's: a buffer load, whose counter the compiler follows exactly
// (a global load into LDS makes it wait for everything under way at the next use of anything). Its offsets have 32 bits.
EIF_DEV void load_lds16(__amdgpu_buffer_rsrc_t src, uint32_t lane_offset, uint32_t offset, void *dst)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void *)dst, 16, lane_offset, offset, 0, 0);
}

// Many token rows: a workgroup of four waves takes 16 TT token rows and 4 RT row tiles, RT to a wave (gated: RT / 2 of the
// gate's and the same of the up projection's). A wave's row tiles are its own, so their codes go from memory straight
// into registers; the token rows are shared, so they go into LDS.
//   PF 1: token rows straight into LDS, one span ahead, and codes by steps of 128 columns, three ahead. PF 3: both three spans
// ahead, token rows through registers; for small tiles, of which a CU has few.
//   A span of a token tile is 16 rows of 128 bytes, 8 pieces h of 16 (piece h = 2 slot + step). A load covers eight rows,
// whole cache lines; row n's piece h lies at place 8 (n % 8) + (h ^ place(n)) of its half of the tile. LDS takes a read of
// 16 bytes a lane 16 lanes at a time, rows 0-3 and 12-15 of one slot with rows 4-11 of the next; place() gives them 16
// different groups of banks (with n / 2 in its place they met in pairs).
//   What bounds it: 4096 rows through 8192x8192 take 126 to 136 us, 4.0 to 4.4 PFLOP/s; the matrix instructions alone run at 7.1 here (at
// 1.7 GHz, where power holds them), and the 134 MB of outputs take 28 us of it. A span of the two workgroups on a CU is 2048
// cycles of matrix instructions, and L2 has to bring 96 KB meanwhile. (Before whole-line loads of token rows and scales by
// pairs of spans its request rate was the bound: 271 us. Tiles of 256x256 rows with eight waves took 5 % longer, a workgroup
// that goes on to the next row block too: nothing covers its waits.)
template <int RT, int TT, int PF, bool GLU, bool GROUPED>
__global__ __launch_bounds__(256, RT * TT <= 32 ? 2 : 1) void mx4_gemm_kernel(Mx4Args a)
{
    constexpr int NT = GLU ? 2 : 1, OT = RT / NT, TM = 16 * TT;
    constexpr int R = PF + 1, SV = R / 2;       // spans in LDS and registers, pairs of spans of scales under way
    constexpr int PT = (2 * TT + 3) / 4;        // half tiles of token rows that a wave stages
    constexpr int PS = (2 * TM + 255) / 256;    // scales that a thread stages: a row's of one span of a pair
    static_assert(PF == 1 || PF == 3, "the loop below goes by four spans");
    // spans in turn; an array each: the compiler then knows that a load into one does not touch a read of the other
    __shared__ v4i xt0[TT * 128], xt1[TT * 128];
    __shared__ __align__(8) uint16_t xs0[TM * 8], xs1[TM * 8];   // pairs of spans in turn: [row][span of the pair][slot]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, slot = lane >> 4;
    const int otiles = GLU ? a.tiles / 2 : a.tiles;
    const int rblocks = (otiles + 4 * OT - 1) / (4 * OT);
    // Workgroups go to the XCDs in turn: each XCD gets a stretch of consecutive ids, ordered in strips of 8 row blocks, so
    // that what it works on at a time is about as many row blocks as groups of token rows, which meet in its L2.
    const unsigned per = (gridDim.x + 7) / 8;
    const unsigned id = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (id >= (unsigned)rblocks * a.groups) return;
    const int strip = id / (8u * a.groups), rest = id % (8u * a.groups), high = min(8, rblocks - 8 * strip);
    const int rb = 8 * strip + rest % high, group = rest / high;
    int expert = 0, lo = group * TM, hi = min(lo + TM, a.M);
    if (GROUPED && !find_group<TM>(a, group, expert, lo, hi)) return;
    const int last = a.spans - 1;

    struct Weights {
        v4i c[RT][2];
        uint32_t s[RT];
    };
    Weights w[PF > 1 ? R : 1];
    v4i ring[PF > 1 ? 1 : 4][RT];        // PF 1: by steps, half a span each
    uint32_t sw[PF > 1 ? 1 : 2][RT];     // pairs of spans in turn
    // Row tiles behind the matrix's last (of the last row block) are read too, the allocation holds enough of them, and not
    // stored. The same for all lanes:
    const uint32_t tile_c = a.spans * 2048u, tile_s = (a.spans + 1) / 2 * 256u;
    const uint8_t *wc[NT];
    const uint8_t *ws[NT];
    // A lane's offset as 32 bits that the compiler does not widen ahead of the loop: the loads take it beside a scalar address,
    // without a 64-bit address register each.
    auto offset = [&](uint32_t bytes) {
        asm volatile("" : "+v"(bytes));
        return bytes;
    };
#pragma unroll
    for (int h = 0; h < NT; ++h) {
        const size_t t = (size_t)expert * a.tiles + h * otiles + (rb * 4 + wave) * OT;
        wc[h] = a.wc + t * tile_c;
        ws[h] = reinterpret_cast<const uint8_t *>(a.ws) + t * tile_s;
    }
    auto load_weights = [&](int p, Weights &f) {
        const uint32_t lane16 = offset(lane * 16u), lane4 = offset(lane * 4u);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const uint8_t *src = wc[i / OT] + (i % OT * tile_c + p * 2048u);
            f.c[i][0] = *reinterpret_cast<const v4i *>(src + lane16);
            f.c[i][1] = *reinterpret_cast<const v4i *>(src + 1024 + lane16);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) f.s[i] = *reinterpret_cast<const uint32_t *>(ws[i / OT] + (i % OT * tile_s + p / 2 * 256u) + lane4);
    };
    auto load_step = [&](int p, int step, v4i *c) {
        const uint32_t lane16 = offset(lane * 16u);
#pragma unroll
        for (int i = 0; i < RT; ++i)
            c[i] = *reinterpret_cast<const v4i *>(wc[i / OT] + (i % OT * tile_c + p * 2048u + step * 1024u) + lane16);
    };
    auto load_pair = [&](int q, uint32_t *v) {
        const uint32_t lane4 = offset(lane * 4u);
#pragma unroll
        for (int i = 0; i < RT; ++i) v[i] = *reinterpret_cast<const uint32_t *>(ws[i / OT] + (i % OT * tile_s + q * 256u) + lane4);
    };
    if constexpr (PF == 1) {
        load_pair(0, sw[0]);
        load_step(0, 0, ring[0]);
        load_step(0, 1, ring[1]);
        load_step(min(1, last), 0, ring[2]);
    } else {
#pragma unroll
        for (int k = 0; k < PF; ++k) load_weights(min(k, last), w[k]);
    }

    auto operand_row = [&](int m) {
        if (m >= hi) return 0;   // row 0 is there to be read; its sums are not stored
        if (!GROUPED) return m;
        const int r = a.index ? a.index[m] : m;
        return r >= 0 && r < a.rows_in ? r : 0;
    };
    // where there are fewer half tiles than waves, or rows than threads, some stage the same
    const int half0 = PT * wave % (2 * TT);
    const uint8_t *xr[PF == 1 ? 1 : PT];
    uint32_t xo[PF == 1 ? PT : 1];
#pragma unroll
    for (int j = 0; j < PT; ++j) {
        const int half = half0 + j, r = 8 * (half & 1) + (lane >> 3);
        const int64_t at = operand_row(lo + 16 * (half >> 1) + r) * a.ldc + ((lane & 7) ^ place(r)) * 16;
        if constexpr (PF == 1)
            xo[j] = (uint32_t)at;   // launch_product sees to it that it fits
        else
            xr[j] = a.codes + at;
    }
    const auto codes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.codes), 0, a.code_bytes, 0x00027000);
    const uint8_t *sr[PS];
#pragma unroll
    for (int j = 0; j < PS; ++j) sr[j] = a.scales + operand_row(lo + (j * 256 + (int)threadIdx.x) % (2 * TM) / 2) * a.lds;
    const int odd_thread = threadIdx.x & 1;
    // PF 1: from memory straight into LDS; 3: through registers, whose loads the compiler waits for one by one
    v4i xv[R][PT];
    auto load_rows = [&](int p, v4i *v, v4i *dst) {
#pragma unroll
        for (int j = 0; j < PT; ++j) {
            if constexpr (PF == 1)
                load_lds16(codes, xo[j], p * 128u, dst + (half0 + j) * 64);
            else
                v[j] = *reinterpret_cast<const v4i *>(xr[j] + (size_t)p * 128);
        }
    };
    auto store_rows = [&](const v4i *v, v4i *dst) {
        if constexpr (PF > 1) {
#pragma unroll
            for (int j = 0; j < PT; ++j) dst[(half0 + j) * 64 + lane] = v[j];
        }
    };
    uint2 sv[SV][PS];
    auto load_scales = [&](int q, uint2 *v) {   // of a pair of spans
#pragma unroll
        for (int j = 0; j < PS; ++j) v[j] = *reinterpret_cast<const uint2 *>(sr[j] + (size_t)min(2 * q + odd_thread, last) * 8);
    };
    auto store_scales = [&](const uint2 *v, uint16_t *dst) {
#pragma unroll
        for (int j = 0; j < PS; ++j) *reinterpret_cast<uint2 *>(&dst[(j * 256 + threadIdx.x) % (2 * TM) * 4]) = v[j];
    };
    // What the waves put into LDS is there. PF 1: this wave's loads into it too, the N loads behind them may be under way.
    // (__syncthreads() would wait for all loads.) Matrix instructions may move past, memory's may not.
    auto arrived = [&](auto newer) {
        constexpr int N = decltype(newer)::value;
        asm volatile("" ::: "memory");
        if constexpr (PF == 1)
            __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4 << 14));   // vmcnt(N) lgkmcnt(0)
        else
            __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0x8);
    };
    v4i *const xt[2] = {xt0, xt1};
    uint16_t *const xs[2] = {xs0, xs1};
#pragma unroll
    for (int q = 0; q < SV; ++q) load_scales(min(q, last / 2), sv[q]);
#pragma unroll
    for (int k = 0; k < PF; ++k) load_rows(min(k, last), xv[k], xt[k & 1]);

    v4f acc[RT][TT] = {};
    // where a piece lies that this lane reads: row n's 2 slot and 2 slot + 1
    const int at0 = 64 * (n >> 3) + 8 * (n & 7) + ((2 * slot) ^ place(n)), at1 = at0 ^ 1;
    // The span p = K modulo 4. What goes out here is for the span p + PF (near the end: the last one, again. Without a
    // branch, so that the compiler knows how many loads are under way and waits for the older ones alone).
    auto span = [&](auto k, int p) {
        constexpr int K = decltype(k)::value, H = K & 1, Q = K >> 1;
        if (H == 0) load_scales(min(p / 2 + SV, last / 2), sv[Q % SV]);
        if constexpr (PF == 1) {
            if (H == 0) load_pair(min(p / 2 + 1, last / 2), sw[Q ^ 1]);
            load_rows(min(p + 1, last), nullptr, xt[H ^ 1]);
            // where the loads stand is where they go out: behind these, and ahead of arrived(), the codes of two steps
            __builtin_amdgcn_sched_barrier(0);
            constexpr int L = 2;   // pieces read ahead
            v4i b[L + 1];
            uint32_t sx[TT];
            auto read = [&](int u) {   // u = step TT + t
                const int t = u % TT;
                b[u % (L + 1)] = xt[H][t * 128 + (u < TT ? at0 : at1)];
                if (u < TT) sx[t] = xs[Q][(n * 2 + H) * 4 + slot + t * 128];
            };
#pragma unroll
            for (int u = 0; u < 2 * TT; ++u) {
                if (u == 0) load_step(min(p + 1, last), 1, ring[(2 * H + 3) % 4]);
                if (u == TT) load_step(min(p + 2, last), 0, ring[2 * H]);
                if (u == 0) {
#pragma unroll
                    for (int l = 0; l < L; ++l) read(l);
                }
                if (u + L < 2 * TT) read(u + L);
                __builtin_amdgcn_sched_barrier(0);
                const int t = u % TT;
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    if (u < TT)
                        acc[i][t] = step_mfma<H, 0>(acc[i][t], ring[2 * H][i], sw[Q][i], b[u % (L + 1)], sx[t]);
                    else
                        acc[i][t] = step_mfma<H, 1>(acc[i][t], ring[2 * H + 1][i], sw[Q][i], b[u % (L + 1)], sx[t]);
                }
            }
        } else {
            constexpr int B = K % R, N = (K + PF) % R;
            load_rows(min(p + PF, last), xv[N], xt[N & 1]);
            load_weights(min(p + PF, last), w[N]);
            __builtin_amdgcn_sched_barrier(0);   // where the loads stand is where they go out
            v4i b[2][2];
            uint32_t sx[2];
            auto read = [&](int t) {
                b[t & 1][0] = xt[H][t * 128 + at0];
                b[t & 1][1] = xt[H][t * 128 + at1];
                sx[t & 1] = xs[Q][(n * 2 + H) * 4 + slot + t * 128];
            };
            read(0);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                if (t + 1 < TT) read(t + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i][t] = span_mfma<H>(acc[i][t], w[B].c[i][0], w[B].c[i][1], w[B].s[i], b[t & 1][0], b[t & 1][1], sx[t & 1]);
            }
            store_rows(xv[(K + 1) % R], xt[H ^ 1]);
        }
        if (H == 1) store_scales(sv[(Q + 1) % SV], xs[Q ^ 1]);
        arrived(std::integral_constant<int, 2 * RT>{});
    };
    store_rows(xv[0], xt0);
    store_scales(sv[0], xs0);
    arrived(std::integral_constant<int, 0>{});
    auto pair = [&](auto q, int p) {
        constexpr int Q = decltype(q)::value;
        span(std::integral_constant<int, 2 * Q>{}, p);
        if (p == last) return;
        span(std::integral_constant<int, 2 * Q + 1>{}, p + 1);
    };
    for (int p = 0; p <= last; p += 4) {
        pair(std::integral_constant<int, 0>{}, p);
        if (p + 2 <= last) pair(std::integral_constant<int, 1>{}, p + 2);
    }

    bool ok[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const int m = lo + 16 * t + n;
        ok[t] = m < hi;
        if (GROUPED) {
            const int c = min(m, hi - 1), r = a.index ? a.index[c] : c;
            ok[t] = ok[t] && r >= 0 && r < a.rows_in;
        }
    }
    const int out_rows = GLU ? a.rows / 2 : a.rows, tile0 = (rb * 4 + wave) * OT;
    if (tile0 >= otiles) return;
    float b0[OT][4] = {}, b1[OT][4] = {};
    if (a.bias) {
        const float *bias = a.bias + (size_t)expert * a.rows;
#pragma unroll
        for (int i = 0; i < OT; ++i) load_bias<GLU>(bias, (tile0 + i) * 16 + slot * 4, out_rows, b0[i], b1[i]);
    }
    auto store = [&](auto whole) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            float *yr = a.y + (int64_t)(lo + 16 * t + n) * a.ldy;
            if constexpr (decltype(whole)::value && OT % 2 == 0) {
                // Two row tiles of a token row are a cache line, but in one lane. Lanes of two token rows exchange a tile
                // each, so that a store covers the lines of eight token rows and not the halves of sixteen; whole lines can
                // go past L2, whose room is the operands' (us, plain stores of halves / of lines / lines past L2: 4096 rows
                // through 8192x8192 150 / 148 / 134, 16384 by expert through 2048x1408 83.7 / 78.6 / 73.8).
                const int odd = n & 1;
                const bool other = __shfl_xor((int)ok[t], 1, 64);
                float *y0 = yr - odd * a.ldy + (tile0 + odd) * 16 + slot * 4, *y1 = y0 + a.ldy;
                const bool ok0 = odd ? other : ok[t], ok1 = odd ? ok[t] : other;
#pragma unroll
                for (int i = 0; i < OT; i += 2) {
                    float u[4], v[4];
                    outputs<GLU>(acc[i][t], acc[RT - OT + i][t], b0[i], b1[i], u);
                    outputs<GLU>(acc[i + 1][t], acc[RT - OT + i + 1][t], b0[i + 1], b1[i + 1], v);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float got = xlane<1>(odd ? u[j] : v[j]);
                        u[j] = odd ? got : u[j];
                        v[j] = odd ? v[j] : got;
                    }
                    if (ok0) __builtin_nontemporal_store((v4f{u[0], u[1], u[2], u[3]}), reinterpret_cast<v4f *>(y0 + i * 16));
                    if (ok1) __builtin_nontemporal_store((v4f{v[0], v[1], v[2], v[3]}), reinterpret_cast<v4f *>(y1 + i * 16));
                }
            } else {
                if (!ok[t]) continue;
#pragma unroll
                for (int i = 0; i < OT; ++i)
                    store_outputs<GLU, decltype(whole)::value>(yr, (tile0 + i) * 16 + slot * 4, out_rows, acc[i][t],
                                                               acc[RT - OT + i][t], b0[i], b1[i]);
            }
        }
    };
    if (a.vec && (tile0 + OT) * 16 <= out_rows)
        store(std::true_type{});
    else
        store(std::false_type{});
}

// ---- host ----

constexpr int64_t kLaunchThreads = UINT32_MAX;   // threads that a launch holds at most
constexpr int64_t kLaunchBlocks = kLaunchThreads / 256;   // workgroups of 256
constexpr int kMaxCols = 1 << 24;
constexpr int kMaxRows = 1 << 30;
constexpr int kMaxExperts = 4096;    // a workgroup of a product by expert goes over all offsets
constexpr int kTilesBehind = 15;   // row tiles that a product may read behind the last
constexpr int kRowsMaxM = 8, kRowsMaxCols = 16384;

inline int spans_of(int cols) { return (cols - 1) / kSpan + 1; }

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <typename T>
int launch_quant(const void *x, int64_t ldx, int rows, int cols, uint8_t *codes, int64_t ldc, uint8_t *scales,
                 int64_t lds, float *values, int64_t ldv, hipStream_t st)
{
    const int spans = spans_of(cols);
    if (((int64_t)rows * spans + 3) / 4 > INT32_MAX) return EIF_HIP_E_LIMIT;
    const bool vec = aligned(x, 4 * sizeof(T)) && ldx % 4 == 0 && cols % 4 == 0, vv = aligned(values, 16) && ldv % 4 == 0;
    const int64_t per = kLaunchBlocks * 4 / spans;   // rows of a launch
    for (int64_t row = 0; row < rows; row += per) {
        const int n = (int)std::min(per, rows - row);
        const unsigned blocks = (unsigned)(((int64_t)n * spans + 3) / 4);
        const T *xt = static_cast<const T *>(x) + row * ldx;
        uint8_t *c = codes ? codes + row * ldc : nullptr, *s = scales ? scales + row * lds : nullptr;
        float *v = values ? values + row * ldv : nullptr;
        if (vec)
            quant_rows_kernel<T, true><<<blocks, 256, 0, st>>>(xt, ldx, n, cols, spans, c, ldc, s, lds, v, ldv, vv);
        else
            quant_rows_kernel<T, false><<<blocks, 256, 0, st>>>(xt, ldx, n, cols, spans, c, ldc, s, lds, v, ldv, vv);
        EIF_HIP_LAUNCHED();
    }
    return EIF_HIP_OK;
}

// What every product checks: the weight, its device, the biases, the output and the gated form's rows.
int check_product(const eif_hip_mx4_weight *w, const float *bias, int glu, const float *y, int64_t ldy, int M)
{
    if (!w || M < 0) return EIF_HIP_E_ARG;
    if (M > kMaxRows) return EIF_HIP_E_LIMIT;
    if (glu && w->rows % 32 != 0) return EIF_HIP_E_LIMIT;
    if (ldy < (glu ? w->rows / 2 : w->rows) || (M > 0 && !y)) return EIF_HIP_E_ARG;
    if (!aligned(y, 4) || !aligned(bias, 4)) return EIF_HIP_E_ARG;
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess) return EIF_HIP_E_DEVICE;
    return dev == w->device ? EIF_HIP_OK : EIF_HIP_E_ARG;
}

int check_operand(const eif_hip_mx4_weight *w, const uint8_t *codes, int64_t ldc, const uint8_t *scales, int64_t lds)
{
    if (!codes || !scales || !aligned(codes, 16) || !aligned(scales, 8)) return EIF_HIP_E_ARG;
    if (ldc < w->spans * 128 || ldc % 16 != 0 || lds < w->spans * 8 || lds % 8 != 0) return EIF_HIP_E_ARG;
    return EIF_HIP_OK;
}

// Bytes that `rows` operand rows' codes span, 0 for 2^32 and more.
uint32_t code_bytes(const eif_hip_mx4_weight *w, int64_t ldc, int rows)
{
    const int64_t row = w->spans * 128;
    if (ldc > UINT32_MAX || (rows - 1) * ldc + row > UINT32_MAX) return 0;
    return (uint32_t)((rows - 1) * ldc + row);
}

Mx4Args weight_args(const eif_hip_mx4_weight *w, const float *bias, float *y, int64_t ldy, int M)
{
    Mx4Args a{};
    a.wc = w->codes, a.ws = w->scales, a.tiles = w->tiles, a.spans = w->spans, a.rows = w->rows, a.cols = w->cols;
    a.bias = bias, a.y = y, a.ldy = ldy, a.M = M, a.experts = w->experts;
    a.vec = aligned(y, 16) && ldy % 4 == 0;
    return a;
}

// Groups of `per` token rows: what the grid holds (by expert: however the rows are spread), and about how many there are.
struct Groups {
    int64_t grid, likely;
};
Groups groups_of(const Mx4Args &a, bool grouped, int per)
{
    const int64_t whole = (int64_t)(a.M - 1) / per + 1;
    if (!grouped) return {whole, whole};
    return {whole + a.experts - 1, std::min<int64_t>(whole + a.experts / 2, a.M)};
}

template <typename X, int TT, int KW, int D>
int launch_split_as(const Mx4Args &a, bool glu, bool grouped, hipStream_t st)
{
    const int64_t blocks = groups_of(a, grouped, 16 * TT).grid * eif_ceil_div(glu ? a.tiles / 2 : a.tiles, 8 / KW);
    if (blocks > kLaunchThreads / 512) return EIF_HIP_E_LIMIT;
    const unsigned g = (unsigned)blocks;
    if constexpr (std::is_void<X>::value) {
        if (glu)
            grouped ? mx4_split_kernel<X, TT, KW, D, true, true><<<g, 512, 0, st>>>(a)
                    : mx4_split_kernel<X, TT, KW, D, true, false><<<g, 512, 0, st>>>(a);
        else
            grouped ? mx4_split_kernel<X, TT, KW, D, false, true><<<g, 512, 0, st>>>(a)
                    : mx4_split_kernel<X, TT, KW, D, false, false><<<g, 512, 0, st>>>(a);
    } else {
        const size_t lds = (size_t)a.M * (a.spans * 128 + 16 + a.spans * 8);
        if (glu)
            mx4_split_kernel<X, TT, KW, D, true, false><<<g, 512, lds, st>>>(a);
        else
            mx4_split_kernel<X, TT, KW, D, false, false><<<g, 512, lds, st>>>(a);
    }
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

template <typename X, int TT, int KW>
int launch_split_deep(const Mx4Args &a, bool glu, bool grouped, hipStream_t st)
{
    const int n = eif_ceil_div(a.spans, KW);   // spans of a wave
    if (n == 1) return launch_split_as<X, TT, KW, 1>(a, glu, grouped, st);
    if constexpr (TT == 1) {
        if (n > 2) return launch_split_as<X, TT, KW, 4>(a, glu, grouped, st);
    }
    return launch_split_as<X, TT, KW, 2>(a, glu, grouped, st);
}

// Waves that share a row tile: as many as keep the launch at 4096 row tiles times waves, 4 a SIMD (the rows form: 3500; each
// workgroup quantises the rows, and more waves a tile are more workgroups). Measured on three sets of inputs in turn, which the
// Infinity Cache holds whole or in part (us, 1 / 2 / 4 / 8 waves): one row, 151936x1024
// 13.9 / 14.1 / 15.2 / 23.1; 8 rows, 8192x8192 19.8 / 11.9 / 9.2 / 8.7, gated 13824x2560 in the rows form 11.0 / 9.8 /
// 9.2 / 11.0; 32 rows by expert, about 22 experts of gated 2816x2560 13.6 / 18.1 / 19.4 / 17.2.
template <typename X, int TT>
int launch_split(const Mx4Args &a, bool glu, bool grouped, hipStream_t st)
{
    const int64_t tiles = groups_of(a, grouped, 16 * TT).likely * a.tiles;
    const int64_t waves = std::is_void<X>::value ? 4096 : 3500;
    int kw = 8;
    while (kw > 1 && (kw > a.spans || tiles * kw > waves)) kw /= 2;
    if (kw == 8) return launch_split_deep<X, TT, 8>(a, glu, grouped, st);
    if (kw == 4) return launch_split_deep<X, TT, 4>(a, glu, grouped, st);
    if (kw == 2) return launch_split_deep<X, TT, 2>(a, glu, grouped, st);
    return launch_split_deep<X, TT, 1>(a, glu, grouped, st);
}

// Workgroups of mx4_gemm_kernel<RT, TT>: row blocks times groups.
template <int RT, int TT>
int64_t gemm_blocks(const Mx4Args &a, bool glu, int64_t groups)
{
    return groups * eif_ceil_div(glu ? a.tiles / 2 : a.tiles, 4 * RT / (glu ? 2 : 1));
}

template <int RT, int TT, int PF>
int launch_gemm(Mx4Args a, bool glu, bool grouped, hipStream_t st)
{
    const int64_t groups = groups_of(a, grouped, 16 * TT).grid, blocks = (gemm_blocks<RT, TT>(a, glu, groups) + 7) / 8 * 8;
    if (blocks > kLaunchBlocks) return EIF_HIP_E_LIMIT;
    a.groups = (int)groups;
    const unsigned g = (unsigned)blocks;
    if (glu)
        grouped ? mx4_gemm_kernel<RT, TT, PF, true, true><<<g, 256, 0, st>>>(a)
                : mx4_gemm_kernel<RT, TT, PF, true, false><<<g, 256, 0, st>>>(a);
    else
        grouped ? mx4_gemm_kernel<RT, TT, PF, false, true><<<g, 256, 0, st>>>(a)
                : mx4_gemm_kernel<RT, TT, PF, false, false><<<g, 256, 0, st>>>(a);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

// The form of a product of quantised rows: the largest tile that still gives the 256 CUs workgroups enough (200; 256; 160); of a few
// rows the split form. By expert a tile of more token rows than an expert has on average is mostly empty. The limits are set by
// these measurements, within 6 % of the best form but for 800 rows through 5120x5120 (23.4, where 256x128 takes 20.8). Measured (us; 256
// rows x 128 tokens / 128x128 / 128x64 / 128x32 three spans ahead / split; in brackets the workgroups of the first three):
//   4096 rows, 8192x8192 133 / 149 / 187 / 291 / 1615 (1024, 2048, 4096); 512, gated 13824x2560 15.0 / 16.2 / 18.5 / 25.1 / 87 (216,
//   432, 864); 800, 5120x5120 20.8 / 23.4 / 23.3 / 26.1 / - (140, 280, 520); 1024, 4096x4096 17.6 / 14.2 / 14.9 / 21.6 / 103 (128,
//   256, 512); 1500, 2560x2560 13.3 / 10.3 / 10.3 / 15.7 / - (120, 240, 480); 384, 8192x8192 29 / 21 / 22 / 29 / - (96, 192, 384);
//   640, 2560x6912 26 / 18.3 / 15.2 / 18.0 / - (50, 100, 200); 128, 8192x8192 29 / 20 / 16.9 / 13.8 / 53 (32, 64, 128); 256,
//   2560x6912 26 / 18.1 / 14.8 / 12.1 / 37 (20, 40, 80); 100, 2560x2560 12.1 / 8.1 / 6.0 / 6.3 / 10.3; 32, 8192x8192 28 / 19 / 16 /
//   13.5 / 15.5; 600, 1024x1024 - / - / 4.3 / 4.2 / 8.2; 60, 4096x1024 - / - / 4.1 / 3.9 / 3.6; 48, 4864x896 7.4 / 5.2 / 4.0 / 4.0 /
//   3.6; 24, 2560x6912 24 / 16 / 14 / 11.6 / 6.1; by expert, gated 2816 rows: 16384 rows to 64 99 / 113 / 121 / 163 / 389, 800 to 32
//   37 / 36 / 30 / 36 / 38; 2048 to 32 of 2048x1408 18.7 / 18.0 / 15.3 / 18.6 / 54.
int launch_product(const Mx4Args &a, bool glu, bool grouped, hipStream_t st)
{
    const int m = grouped ? (a.M - 1) / a.experts + 1 : a.M;   // token rows of a matrix
    if (m <= 16) return launch_split<void, 1>(a, glu, grouped, st);
    const int64_t g128 = groups_of(a, grouped, 128).likely, g64 = groups_of(a, grouped, 64).likely;
    const bool wide = m >= 96 && gemm_blocks<4, 8>(a, glu, g128) >= 200, middle = m >= 96 && gemm_blocks<2, 8>(a, glu, g128) >= 256;
    const bool narrow = gemm_blocks<2, 4>(a, glu, g64) >= 160;
    const int64_t small = gemm_blocks<2, 2>(a, glu, groups_of(a, grouped, 32).likely);
    if (!wide && !middle && !narrow && (small < 64 || small * a.spans < 400))
        return m <= 32 ? launch_split<void, 2>(a, glu, grouped, st) : launch_split<void, 1>(a, glu, grouped, st);
    // The tiles add up in the same order, so that this one can take the place of those whose loads have 32-bit offsets without a bit's
    // difference.
    if (a.code_bytes == 0) return launch_gemm<2, 2, 3>(a, glu, grouped, st);
    if (wide) return launch_gemm<4, 8, 1>(a, glu, grouped, st);
    if (middle) return launch_gemm<2, 8, 1>(a, glu, grouped, st);
    return narrow ? launch_gemm<2, 4, 1>(a, glu, grouped, st) : launch_gemm<2, 2, 3>(a, glu, grouped, st);
}

}  // namespace

extern "C" {

int eif_hip_mx4_kpad(int cols) { return cols < 1 || cols > kMaxCols ? 0 : spans_of(cols) * kSpan; }

int eif_hip_mx4_quant_rows(const void *x, int type, int64_t ldx, int rows, int cols, uint8_t *codes, int64_t ldc,
                           uint8_t *scales, int64_t lds, float *values, int64_t ldv, void *stream)
{
    if (rows < 0 || cols < 1 || ldx < cols || type < EIF_HIP_F32 || type > EIF_HIP_BF16) return EIF_HIP_E_ARG;
    if (cols > kMaxCols) return EIF_HIP_E_LIMIT;
    const int64_t spans = spans_of(cols);
    if (!codes != !scales || (!codes && !values)) return EIF_HIP_E_ARG;
    if (codes && (ldc < spans * 128 || ldc % 16 != 0 || lds < spans * 8 || lds % 8 != 0 || !aligned(codes, 16) || !aligned(scales, 8)))
        return EIF_HIP_E_ARG;
    if (values && ldv < cols) return EIF_HIP_E_ARG;
    if (rows == 0) return EIF_HIP_OK;
    if (!x || !aligned(x, type == EIF_HIP_F32 ? 4 : 2) || !aligned(values, 4)) return EIF_HIP_E_ARG;
    hipStream_t st = (hipStream_t)stream;
    if (type == EIF_HIP_F32) return launch_quant<float>(x, ldx, rows, cols, codes, ldc, scales, lds, values, ldv, st);
    if (type == EIF_HIP_F16) return launch_quant<__half>(x, ldx, rows, cols, codes, ldc, scales, lds, values, ldv, st);
    return launch_quant<__hip_bfloat16>(x, ldx, rows, cols, codes, ldc, scales, lds, values, ldv, st);
}

int eif_hip_mx4_weight_create(eif_hip_mx4_weight **out, int experts, int rows, int cols, const uint8_t *codes,
                              int64_t ldc, const uint8_t *scales, int64_t lds, int src_on_device, void *stream)
{
    if (!out) return EIF_HIP_E_ARG;
    *out = nullptr;
    if (!codes || !scales || experts < 1 || rows < 1 || cols < 1) return EIF_HIP_E_ARG;
    if (ldc < ((int64_t)cols + 1) / 2 || lds < ((int64_t)cols + 31) / 32) return EIF_HIP_E_ARG;
    if (cols > kMaxCols || rows > kMaxRows || experts > kMaxExperts) return EIF_HIP_E_LIMIT;
    eif_hip_mx4_weight q{};
    q.experts = experts, q.rows = rows, q.cols = cols, q.tiles = eif_ceil_div(rows, 16), q.spans = spans_of(cols);
    if ((int64_t)experts * q.tiles > INT32_MAX) return EIF_HIP_E_LIMIT;
    if (hipGetDevice(&q.device) != hipSuccess) return EIF_HIP_E_DEVICE;
    const size_t tiles = (size_t)experts * q.tiles;
    const size_t cbytes = tiles * tile_codes(q.spans), sdwords = tiles * tile_scales(q.spans);
    const size_t pieces = cbytes / 16, per = (size_t)kLaunchBlocks * 256;   // of a launch
    hipStream_t st = (hipStream_t)stream;
    // host rows go up as they lie, up to the last row's end
    const size_t all = (size_t)experts * rows;
    if (ldc > INT64_MAX / (int64_t)all || lds > INT64_MAX / (int64_t)all) return EIF_HIP_E_LIMIT;
    const size_t src_c = (all - 1) * ldc + ((size_t)cols + 1) / 2, src_s = (all - 1) * lds + ((size_t)cols + 31) / 32;
    uint8_t *up = nullptr;
    int rc = EIF_HIP_OK;
    const size_t codes_all = cbytes + kTilesBehind * tile_codes(q.spans);
    q.bytes = codes_all + (sdwords + kTilesBehind * tile_scales(q.spans)) * 4;
    if (hipMalloc(&q.codes, q.bytes) != hipSuccess || (!src_on_device && hipMalloc(&up, src_c + src_s) != hipSuccess)) {
        (void)hipGetLastError();
        rc = EIF_HIP_E_NOMEM;
    }
    if (rc == EIF_HIP_OK) q.scales = reinterpret_cast<uint32_t *>(q.codes + codes_all);   // one allocation
    if (rc == EIF_HIP_OK && !src_on_device) {
        if (hipMemcpyAsync(up, codes, src_c, hipMemcpyHostToDevice, st) != hipSuccess ||
            hipMemcpyAsync(up + src_c, scales, src_s, hipMemcpyHostToDevice, st) != hipSuccess)
            rc = EIF_HIP_E_DEVICE;
        codes = up, scales = up + src_c;
    }
    const bool vec = aligned(codes, 16) && ldc % 16 == 0;
    for (size_t i = 0; i < pieces && rc == EIF_HIP_OK; i += per) {
        const unsigned blocks = (unsigned)((std::min(per, pieces - i) + 255) / 256);
        mx4_repack_kernel<<<blocks, 256, 0, st>>>(codes, ldc, rows, cols, q.tiles, q.spans, q.codes, i, pieces, vec);
        if (hipGetLastError() != hipSuccess) rc = EIF_HIP_E_DEVICE;
    }
    for (size_t i = 0; i < sdwords && rc == EIF_HIP_OK; i += per) {
        const unsigned blocks = (unsigned)((std::min(per, sdwords - i) + 255) / 256);
        mx4_repack_scales_kernel<<<blocks, 256, 0, st>>>(scales, lds, rows, cols, q.tiles, q.spans, q.scales, i, sdwords);
        if (hipGetLastError() != hipSuccess) rc = EIF_HIP_E_DEVICE;
    }
    if (rc != EIF_HIP_E_NOMEM && hipStreamSynchronize(st) != hipSuccess && rc == EIF_HIP_OK) rc = EIF_HIP_E_DEVICE;
    if (up) (void)hipFree(up);
    eif_hip_mx4_weight *h = rc == EIF_HIP_OK ? new (std::nothrow) eif_hip_mx4_weight(q) : nullptr;
    if (!h) {
        if (q.codes) (void)hipFree(q.codes);
        return rc == EIF_HIP_OK ? EIF_HIP_E_NOMEM : rc;
    }
    *out = h;
    return EIF_HIP_OK;
}

void eif_hip_mx4_weight_destroy(eif_hip_mx4_weight *w)
{
    if (!w) return;
    (void)hipFree(w->codes);
    delete w;
}

int eif_hip_mx4_weight_info(const eif_hip_mx4_weight *w, int *experts, int *rows, int *cols, int *kpad, size_t *bytes)
{
    if (!w) return EIF_HIP_E_ARG;
    if (experts) *experts = w->experts;
    if (rows) *rows = w->rows;
    if (cols) *cols = w->cols;
    if (kpad) *kpad = w->spans * kSpan;
    if (bytes) *bytes = w->bytes;
    return EIF_HIP_OK;
}

int eif_hip_mx4_linear(const eif_hip_mx4_weight *w, const uint8_t *codes, int64_t ldc, const uint8_t *scales, int64_t lds,
                       const float *bias, int glu, float *y, int64_t ldy, int M, void *stream)
{
    int rc = check_product(w, bias, glu, y, ldy, M);
    if (rc) return rc;
    if (w->experts != 1) return EIF_HIP_E_ARG;
    if (M == 0) return EIF_HIP_OK;
    if ((rc = check_operand(w, codes, ldc, scales, lds)) != 0) return rc;
    Mx4Args a = weight_args(w, bias, y, ldy, M);
    a.codes = codes, a.ldc = ldc, a.scales = scales, a.lds = lds;
    a.code_bytes = code_bytes(w, ldc, M);
    return launch_product(a, glu, false, (hipStream_t)stream);
}

int eif_hip_mx4_linear_rows(const eif_hip_mx4_weight *w, const void *x, int type, int64_t ldx, const float *bias, int glu,
                            float *y, int64_t ldy, int M, void *stream)
{
    const int rc = check_product(w, bias, glu, y, ldy, M);
    if (rc) return rc;
    if (w->experts != 1 || ldx < w->cols || type < EIF_HIP_F32 || type > EIF_HIP_BF16) return EIF_HIP_E_ARG;
    if (M > kRowsMaxM || w->cols > kRowsMaxCols) return EIF_HIP_E_LIMIT;
    if (M == 0) return EIF_HIP_OK;
    if (!x || !aligned(x, type == EIF_HIP_F32 ? 4 : 2)) return EIF_HIP_E_ARG;
    Mx4Args a = weight_args(w, bias, y, ldy, M);
    a.x = x, a.ldx = ldx;
    hipStream_t st = (hipStream_t)stream;
    a.vecx = aligned(x, type == EIF_HIP_F32 ? 16 : 8) && ldx % 4 == 0 && w->cols % 4 == 0;
    if (type == EIF_HIP_F32) return launch_split<float, 1>(a, glu, false, st);
    return type == EIF_HIP_F16 ? launch_split<__half, 1>(a, glu, false, st) : launch_split<__hip_bfloat16, 1>(a, glu, false, st);
}

int eif_hip_mx4_linear_grouped(const eif_hip_mx4_weight *w, const uint8_t *codes, int64_t ldc, const uint8_t *scales,
                               int64_t lds, int rows_in, const int32_t *row_index, const int32_t *offsets,
                               const float *bias, int glu, float *y, int64_t ldy, int M, void *stream)
{
    int rc = check_product(w, bias, glu, y, ldy, M);
    if (rc) return rc;
    if (rows_in < 0) return EIF_HIP_E_ARG;
    if (M == 0 || rows_in == 0) return EIF_HIP_OK;
    if ((rc = check_operand(w, codes, ldc, scales, lds)) != 0) return rc;
    if (!offsets || !aligned(offsets, 4) || !aligned(row_index, 4)) return EIF_HIP_E_ARG;
    Mx4Args a = weight_args(w, bias, y, ldy, M);
    a.codes = codes, a.ldc = ldc, a.scales = scales, a.lds = lds;
    a.rows_in = rows_in, a.index = row_index, a.offsets = offsets;
    a.code_bytes = code_bytes(w, ldc, rows_in);
    return launch_product(a, glu, true, (hipStream_t)stream);
}

}  // extern "C"
