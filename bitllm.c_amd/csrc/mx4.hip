// mx4.hip -- microscaled 4-bit (MXFP4) operators: quantisation of rows, resident matrices, products (eif_hip_mx.h).
#include "hip_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <new>

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

// One wave a row and span: lane l has columns 4 l .. 4 l + 3, a block is eight lanes.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T *x, int64_t ldx, int rows, int cols, int spans,
                                                         uint8_t *codes, int64_t ldc, uint8_t *scales, int64_t lds,
                                                         float *values, int64_t ldv)
{
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t row = unit / spans;
    const int span = (int)(unit % spans), c = span * kSpan + lane * 4;
    if (row >= rows) return;
    const T *xr = x + row * ldx;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (VEC && c + 4 <= cols) {
        const Quad<T> q = *reinterpret_cast<const Quad<T> *>(xr + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32(q.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < cols) v[i] = to_f32(xr[c + i]);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = umax(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = umax(m, __float_as_uint(xlane<1>(__uint_as_float(m))));
    m = umax(m, __float_as_uint(xlane<2>(__uint_as_float(m))));
    m = umax(m, __float_as_uint(xlane<4>(__uint_as_float(m))));
    const uint32_t b = scale_byte(m);
    const uint32_t q = codes4(v, scale_inverse(b), b != 255);
    if (codes) {
        *reinterpret_cast<uint16_t *>(codes + row * ldc + (c >> 1)) = (uint16_t)q;
        if ((lane & 7) == 0) scales[row * lds + (c >> 5)] = (uint8_t)b;
    }
    if (values) {
        const float s = scale_value(b);
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
        const float o[4] = {lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
        float *vr = values + row * ldv;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < cols) vr[c + i] = o[i];
    }
}

// ---- the resident layout ----

// One thread a 16-byte piece of the layout: its lane's row, block and step.
__global__ __launch_bounds__(256) void mx4_repack_kernel(const uint8_t *src, int64_t ldc, int rows, int cols, int tiles,
                                                         int spans, uint8_t *dst, size_t pieces)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
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
        for (int j = 0; j < 16; ++j) {
            const int c = c0 + 2 * j;
            uint32_t v = c < cols ? s[c >> 1] : 0;
            if (c + 1 >= cols) v &= 0x0F;   // the last byte of an odd count holds one code
            w[j >> 2] |= v << (8 * (j & 3));
        }
    }
    reinterpret_cast<uint4 *>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

// One thread a dword of scales: the lane's four blocks of a pair of spans.
__global__ __launch_bounds__(256) void mx4_repack_scales_kernel(const uint8_t *src, int64_t lds, int rows, int cols,
                                                                int tiles, int spans, uint32_t *dst, size_t n)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
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
    // by expert
    int experts, rows_in;
    const int32_t *index, *offsets;
    // rows form
    const void *x;
    int64_t ldx;
    int cols;
};

// Two MFMAs of one span: codes c0, c1 of a row tile, their scales in bytes 2 h, 2 h + 1 of sw; operand rows' in bytes
// 0, 1 of sx.
template <int H>
EIF_DEV v4f span_mfma(v4f acc, v4i w0, v4i w1, uint32_t sw, v4i x0, v4i x1, uint32_t sx)
{
    const v8i a0 = {w0[0], w0[1], w0[2], w0[3], 0, 0, 0, 0}, a1 = {w1[0], w1[1], w1[2], w1[3], 0, 0, 0, 0};
    const v8i b0 = {x0[0], x0[1], x0[2], x0[3], 0, 0, 0, 0}, b1 = {x1[0], x1[1], x1[2], x1[3], 0, 0, 0, 0};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a0, b0, acc, 4, 4, 2 * H, (int)sw, 0, (int)sx);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a1, b1, acc, 4, 4, 2 * H + 1, (int)sw, 1, (int)sx);
}

EIF_DEV float swiglu(float g, float u) { return (g * (1.0f / (1.0f + expf(-g)))) * u; }

// The g-th group of TM token rows over the experts' ranges: its expert and its rows [lo, hi); false beyond the last.
// One wave's lanes take 64 experts at a time; a range is cut to [0, M], so every row is in bounds whatever the offsets.
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
            expert = e0 + l;
            lo = s0 + at * TM;
            hi = min(lo + TM, s0 + n0);
            return true;
        }
        base += __shfl(sum, 63, 64);
    }
    return false;
}

// One workgroup a row tile (gated: the gate's and the up projection's) and 16 TT token rows; its four waves take the pairs
// of spans in turn and add their sums up in LDS.
template <int TT, bool GLU, bool GROUPED>
__global__ __launch_bounds__(256) void mx4_linear_kernel(Mx4Args a)
{
    constexpr int NT = GLU ? 2 : 1, TM = 16 * TT;
    __shared__ v4f red[4][NT * TT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, slot = lane >> 4;
    const int otiles = GLU ? a.tiles / 2 : a.tiles;
    const int tile = blockIdx.x % otiles, group = blockIdx.x / otiles;
    int expert = 0, lo = group * TM, hi = min(lo + TM, a.M);
    if (GROUPED && !find_group<TM>(a, group, expert, lo, hi)) return;

    const uint8_t *xr[TT];
    const uint8_t *sr[TT];
    bool ok[TT];
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
    v4f acc[NT][TT] = {};
    const size_t first = (size_t)expert * a.tiles + tile;
    const uint8_t *wc[NT];
    const uint32_t *ws[NT];
#pragma unroll
    for (int h = 0; h < NT; ++h) {
        wc[h] = a.wc + (first + h * otiles) * tile_codes(a.spans) + lane * 16;
        ws[h] = a.ws + (first + h * otiles) * tile_scales(a.spans) + lane;
    }
    for (int q = wave; 2 * q < a.spans; q += 4) {
        uint32_t sw[NT];
#pragma unroll
        for (int h = 0; h < NT; ++h) sw[h] = ws[h][(size_t)q * 64];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int p = 2 * q + s;
            if (p >= a.spans) break;
            v4i w[NT][2];
#pragma unroll
            for (int h = 0; h < NT; ++h) {
                w[h][0] = *reinterpret_cast<const v4i *>(wc[h] + (size_t)p * 2048);
                w[h][1] = *reinterpret_cast<const v4i *>(wc[h] + (size_t)p * 2048 + 1024);
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const v4i x0 = *reinterpret_cast<const v4i *>(xr[t] + (size_t)p * 128);
                const v4i x1 = *reinterpret_cast<const v4i *>(xr[t] + (size_t)p * 128 + 16);
                const uint32_t sx = *reinterpret_cast<const uint16_t *>(sr[t] + p * 8);
#pragma unroll
                for (int h = 0; h < NT; ++h)
                    acc[h][t] = s == 0 ? span_mfma<0>(acc[h][t], w[h][0], w[h][1], sw[h], x0, x1, sx)
                                       : span_mfma<1>(acc[h][t], w[h][0], w[h][1], sw[h], x0, x1, sx);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int t = 0; t < TT; ++t) red[wave][h * TT + t][lane] = acc[h][t];
    __syncthreads();
    const int out_rows = GLU ? a.rows / 2 : a.rows;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        if (t % 4 != wave || !ok[t]) continue;
        v4f s[NT];
#pragma unroll
        for (int h = 0; h < NT; ++h)
            s[h] = ((red[0][h * TT + t][lane] + red[1][h * TT + t][lane]) + red[2][h * TT + t][lane]) + red[3][h * TT + t][lane];
        float *yr = a.y + (int64_t)(lo + 16 * t + n) * a.ldy;
        const float *bias = a.bias ? a.bias + (size_t)expert * a.rows : nullptr;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = tile * 16 + slot * 4 + i;
            if (r >= out_rows) continue;
            float v = s[0][i] + (bias ? bias[r] : 0.0f);
            if (GLU) v = swiglu(v, s[NT - 1][i] + (bias ? bias[out_rows + r] : 0.0f));
            yr[r] = v;
        }
    }
}

// The rows form: every workgroup quantises the token rows into LDS, then takes a row tile as above.
template <typename T, bool GLU>
__global__ __launch_bounds__(256) void mx4_rows_kernel(Mx4Args a)
{
    constexpr int NT = GLU ? 2 : 1;
    __shared__ v4f red[4][NT][64];
    extern __shared__ __align__(16) uint8_t staged[];   // codes [M][ldq], then scales [M][kpad / 32]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, slot = lane >> 4;
    const int otiles = GLU ? a.tiles / 2 : a.tiles, tile = blockIdx.x;
    const int ldq = a.spans * 128 + 16;   // 16 bytes on from row to row in the banks
    uint8_t *sc = staged + a.M * ldq;
    for (int u = wave; u < a.M * a.spans; u += 4) {
        const int row = u / a.spans, c = (u % a.spans) * kSpan + lane * 4;
        const T *xr = static_cast<const T *>(a.x) + row * a.ldx;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < a.cols) v[i] = to_f32(xr[c + i]);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = umax(m, __float_as_uint(v[i]) & 0x7fffffffu);
        m = umax(m, __float_as_uint(xlane<1>(__uint_as_float(m))));
        m = umax(m, __float_as_uint(xlane<2>(__uint_as_float(m))));
        m = umax(m, __float_as_uint(xlane<4>(__uint_as_float(m))));
        const uint32_t b = scale_byte(m);
        const uint32_t q = codes4(v, scale_inverse(b), b != 255);
        *reinterpret_cast<uint16_t *>(staged + row * ldq + (c >> 1)) = (uint16_t)q;
        if ((lane & 7) == 0) sc[row * a.spans * 8 + (c >> 5)] = (uint8_t)b;
    }
    __syncthreads();
    const int row = n < a.M ? n : 0;
    const uint8_t *xr = staged + row * ldq + slot * 32;
    const uint8_t *sr = sc + row * a.spans * 8 + slot * 2;
    v4f acc[NT] = {};
    for (int q = wave; 2 * q < a.spans; q += 4) {
#pragma unroll
        for (int h = 0; h < NT; ++h) {
            const size_t t = tile + h * otiles;
            const uint32_t sw = a.ws[t * tile_scales(a.spans) + (size_t)q * 64 + lane];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int p = 2 * q + s;
                if (p >= a.spans) break;
                const uint8_t *wp = a.wc + t * tile_codes(a.spans) + (size_t)p * 2048 + lane * 16;
                const v4i w0 = *reinterpret_cast<const v4i *>(wp), w1 = *reinterpret_cast<const v4i *>(wp + 1024);
                const v4i x0 = *reinterpret_cast<const v4i *>(xr + p * 128);
                const v4i x1 = *reinterpret_cast<const v4i *>(xr + p * 128 + 16);
                const uint32_t sx = *reinterpret_cast<const uint16_t *>(sr + p * 8);
                acc[h] = s == 0 ? span_mfma<0>(acc[h], w0, w1, sw, x0, x1, sx) : span_mfma<1>(acc[h], w0, w1, sw, x0, x1, sx);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < NT; ++h) red[wave][h][lane] = acc[h];
    __syncthreads();
    if (wave != 0 || n >= a.M) return;
    const int out_rows = GLU ? a.rows / 2 : a.rows;
    v4f s[NT];
#pragma unroll
    for (int h = 0; h < NT; ++h) s[h] = ((red[0][h][lane] + red[1][h][lane]) + red[2][h][lane]) + red[3][h][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = tile * 16 + slot * 4 + i;
        if (r >= out_rows) continue;
        float v = s[0][i] + (a.bias ? a.bias[r] : 0.0f);
        if (GLU) v = swiglu(v, s[NT - 1][i] + (a.bias ? a.bias[out_rows + r] : 0.0f));
        a.y[(int64_t)n * a.ldy + r] = v;
    }
}

// ---- host ----

constexpr int kMaxCols = 1 << 30;
constexpr int kRowsMaxM = 8, kRowsMaxCols = 16384;

inline int spans_of(int cols) { return (cols - 1) / kSpan + 1; }

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <typename T>
int launch_quant(const void *x, int64_t ldx, int rows, int cols, uint8_t *codes, int64_t ldc, uint8_t *scales,
                 int64_t lds, float *values, int64_t ldv, hipStream_t st)
{
    const int spans = spans_of(cols);
    const int64_t blocks = ((int64_t)rows * spans + 3) / 4;
    if (blocks > INT32_MAX) return EIF_HIP_E_LIMIT;
    const T *xt = static_cast<const T *>(x);
    if (aligned(x, 4 * sizeof(T)) && ldx % 4 == 0)
        quant_rows_kernel<T, true><<<(unsigned)blocks, 256, 0, st>>>(xt, ldx, rows, cols, spans, codes, ldc, scales, lds, values, ldv);
    else
        quant_rows_kernel<T, false><<<(unsigned)blocks, 256, 0, st>>>(xt, ldx, rows, cols, spans, codes, ldc, scales, lds, values, ldv);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

// What every product checks: the weight, its device, the output and the gated form's rows.
int check_product(const eif_hip_mx4_weight *w, int glu, const float *y, int64_t ldy, int M)
{
    if (!w || M < 0) return EIF_HIP_E_ARG;
    if (glu && w->rows % 32 != 0) return EIF_HIP_E_LIMIT;
    if (ldy < (glu ? w->rows / 2 : w->rows) || (M > 0 && !y)) return EIF_HIP_E_ARG;
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

Mx4Args weight_args(const eif_hip_mx4_weight *w, const float *bias, float *y, int64_t ldy, int M)
{
    Mx4Args a{};
    a.wc = w->codes, a.ws = w->scales, a.tiles = w->tiles, a.spans = w->spans, a.rows = w->rows, a.cols = w->cols;
    a.bias = bias, a.y = y, a.ldy = ldy, a.M = M, a.experts = w->experts;
    return a;
}

template <int TT>
int launch_linear(const Mx4Args &a, bool glu, bool grouped, hipStream_t st)
{
    const int64_t groups = (int64_t)(a.M - 1) / (16 * TT) + 1 + (grouped ? a.experts - 1 : 0);
    const int64_t blocks = groups * (glu ? a.tiles / 2 : a.tiles);
    if (blocks > INT32_MAX) return EIF_HIP_E_LIMIT;
    const unsigned g = (unsigned)blocks;
    if (glu)
        grouped ? mx4_linear_kernel<TT, true, true><<<g, 256, 0, st>>>(a) : mx4_linear_kernel<TT, true, false><<<g, 256, 0, st>>>(a);
    else
        grouped ? mx4_linear_kernel<TT, false, true><<<g, 256, 0, st>>>(a) : mx4_linear_kernel<TT, false, false><<<g, 256, 0, st>>>(a);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

template <typename T>
int launch_rows(const Mx4Args &a, bool glu, hipStream_t st)
{
    const size_t lds = (size_t)a.M * (a.spans * 128 + 16 + a.spans * 8);
    if (glu)
        mx4_rows_kernel<T, true><<<a.tiles / 2, 256, lds, st>>>(a);
    else
        mx4_rows_kernel<T, false><<<a.tiles, 256, lds, st>>>(a);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
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
    if (cols > kMaxCols || rows > kMaxCols) return EIF_HIP_E_LIMIT;
    eif_hip_mx4_weight q{};
    q.experts = experts, q.rows = rows, q.cols = cols, q.tiles = eif_ceil_div(rows, 16), q.spans = spans_of(cols);
    if ((int64_t)experts * q.tiles > INT32_MAX) return EIF_HIP_E_LIMIT;
    if (hipGetDevice(&q.device) != hipSuccess) return EIF_HIP_E_DEVICE;
    const size_t tiles = (size_t)experts * q.tiles;
    const size_t cbytes = tiles * tile_codes(q.spans), sdwords = tiles * tile_scales(q.spans);
    const size_t pieces = cbytes / 16;
    if (pieces > (size_t)INT32_MAX * 256) return EIF_HIP_E_LIMIT;
    hipStream_t st = (hipStream_t)stream;
    // host rows go up as they lie, up to the last row's end
    const size_t all = (size_t)experts * rows;
    const size_t src_c = (all - 1) * ldc + ((size_t)cols + 1) / 2, src_s = (all - 1) * lds + ((size_t)cols + 31) / 32;
    uint8_t *up = nullptr;
    int rc = EIF_HIP_OK;
    if (hipMalloc(&q.codes, cbytes) != hipSuccess || hipMalloc(&q.scales, sdwords * 4) != hipSuccess ||
        (!src_on_device && hipMalloc(&up, src_c + src_s) != hipSuccess)) {
        (void)hipGetLastError();
        rc = EIF_HIP_E_NOMEM;
    }
    if (rc == EIF_HIP_OK && !src_on_device) {
        if (hipMemcpyAsync(up, codes, src_c, hipMemcpyHostToDevice, st) != hipSuccess ||
            hipMemcpyAsync(up + src_c, scales, src_s, hipMemcpyHostToDevice, st) != hipSuccess)
            rc = EIF_HIP_E_DEVICE;
        codes = up, scales = up + src_c;
    }
    if (rc == EIF_HIP_OK) {
        mx4_repack_kernel<<<(unsigned)((pieces + 255) / 256), 256, 0, st>>>(codes, ldc, rows, cols, q.tiles, q.spans, q.codes, pieces);
        if (hipGetLastError() != hipSuccess) rc = EIF_HIP_E_DEVICE;
    }
    if (rc == EIF_HIP_OK) {
        mx4_repack_scales_kernel<<<(unsigned)((sdwords + 255) / 256), 256, 0, st>>>(scales, lds, rows, cols, q.tiles, q.spans, q.scales, sdwords);
        if (hipGetLastError() != hipSuccess) rc = EIF_HIP_E_DEVICE;
    }
    if (rc != EIF_HIP_E_NOMEM && hipStreamSynchronize(st) != hipSuccess && rc == EIF_HIP_OK) rc = EIF_HIP_E_DEVICE;
    if (up) (void)hipFree(up);
    q.bytes = cbytes + sdwords * 4;
    eif_hip_mx4_weight *h = rc == EIF_HIP_OK ? new (std::nothrow) eif_hip_mx4_weight(q) : nullptr;
    if (!h) {
        if (q.codes) (void)hipFree(q.codes);
        if (q.scales) (void)hipFree(q.scales);
        return rc == EIF_HIP_OK ? EIF_HIP_E_NOMEM : rc;
    }
    *out = h;
    return EIF_HIP_OK;
}

void eif_hip_mx4_weight_destroy(eif_hip_mx4_weight *w)
{
    if (!w) return;
    (void)hipFree(w->codes);
    (void)hipFree(w->scales);
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
    int rc = check_product(w, glu, y, ldy, M);
    if (rc) return rc;
    if (w->experts != 1) return EIF_HIP_E_ARG;
    if (M == 0) return EIF_HIP_OK;
    if ((rc = check_operand(w, codes, ldc, scales, lds)) != 0) return rc;
    Mx4Args a = weight_args(w, bias, y, ldy, M);
    a.codes = codes, a.ldc = ldc, a.scales = scales, a.lds = lds;
    return M <= 16 ? launch_linear<1>(a, glu, false, (hipStream_t)stream) : launch_linear<4>(a, glu, false, (hipStream_t)stream);
}

int eif_hip_mx4_linear_rows(const eif_hip_mx4_weight *w, const void *x, int type, int64_t ldx, const float *bias, int glu,
                            float *y, int64_t ldy, int M, void *stream)
{
    const int rc = check_product(w, glu, y, ldy, M);
    if (rc) return rc;
    if (w->experts != 1 || ldx < w->cols || type < EIF_HIP_F32 || type > EIF_HIP_BF16) return EIF_HIP_E_ARG;
    if (M > kRowsMaxM || w->cols > kRowsMaxCols) return EIF_HIP_E_LIMIT;
    if (M == 0) return EIF_HIP_OK;
    if (!x || !aligned(x, type == EIF_HIP_F32 ? 4 : 2)) return EIF_HIP_E_ARG;
    Mx4Args a = weight_args(w, bias, y, ldy, M);
    a.x = x, a.ldx = ldx;
    hipStream_t st = (hipStream_t)stream;
    if (type == EIF_HIP_F32) return launch_rows<float>(a, glu, st);
    return type == EIF_HIP_F16 ? launch_rows<__half>(a, glu, st) : launch_rows<__hip_bfloat16>(a, glu, st);
}

int eif_hip_mx4_linear_grouped(const eif_hip_mx4_weight *w, const uint8_t *codes, int64_t ldc, const uint8_t *scales,
                               int64_t lds, int rows_in, const int32_t *row_index, const int32_t *offsets,
                               const float *bias, int glu, float *y, int64_t ldy, int M, void *stream)
{
    int rc = check_product(w, glu, y, ldy, M);
    if (rc) return rc;
    if (rows_in < 0) return EIF_HIP_E_ARG;
    if (M == 0 || rows_in == 0) return EIF_HIP_OK;
    if ((rc = check_operand(w, codes, ldc, scales, lds)) != 0) return rc;
    if (!offsets || !aligned(offsets, 4) || !aligned(row_index, 4)) return EIF_HIP_E_ARG;
    Mx4Args a = weight_args(w, bias, y, ldy, M);
    a.codes = codes, a.ldc = ldc, a.scales = scales, a.lds = lds;
    a.rows_in = rows_in, a.index = row_index, a.offsets = offsets;
    return M <= 16 * (int64_t)w->experts ? launch_linear<1>(a, glu, true, (hipStream_t)stream)
                                         : launch_linear<4>(a, glu, true, (hipStream_t)stream);
}

}  // extern "C"
