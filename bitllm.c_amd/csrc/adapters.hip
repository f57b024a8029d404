// adapters.hip -- low-rank adapters of many requests beside a shared projection (eif_hip_adapters.h).
#include "hip_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>

#include "../../include/eif_hip_adapters.h"

// Resident: per slot A, then B, of the adapters' type, zeros beyond rank, cols and rows, each in the order in which a wave reads it:
//   A [16 ranks][32 columns][lane][8]: lane l has rank l % 16 of the 16 and columns 8 (l / 16) .. + 7 of the 32;
//   B [16 rows][lane][16 ranks][4]: lane l has row l % 16 of the 16 and ranks 4 (l / 16) .. + 3 of each 16.
// These are operands of the matrix instructions, and the sums of the first product (ranks 4 (l / 16) .. + 3 in lane l) those of the second.
// And a rank (0: empty) and scale.
struct AdapterMeta {
    int rank;
    float scale;
};
struct eif_hip_adapters {
    char *data;
    AdapterMeta *meta;
    int device, slots, rows, cols, max_rank, type;
    int rank_pad, cols_pad, rows_pad;
    size_t slot_bytes, bytes;
};

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kMaxSlots = 65536, kMaxRank = 256, kMaxDim = 1 << 20, kMaxM = 1 << 24;
constexpr int kColsPad = 32, kRowsPad = 16, kRankPad = 16;

inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline size_t type_size(int type) { return type == EIF_HIP_F32 ? 4 : 2; }

EIF_DEV float to_f32(float v) { return v; }
EIF_DEV float to_f32(__half v) { return __half2float(v); }
EIF_DEV float to_f32(__hip_bfloat16 v) { return __bfloat162float(v); }

template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack { T v[N]; };

template <int N, typename T>
EIF_DEV Pack<T, N> load(const T *p) { return *reinterpret_cast<const Pack<T, N> *>(p); }

// Columns c .. c + 7 of a token row, zeros behind the last. VEC: rows start at 16 bytes, their columns are a multiple of eight.
template <bool VEC, typename T>
EIF_DEV Pack<T, 8> x_pack(const T *xr, int c, int cols)
{
    Pack<T, 8> p;
    if constexpr (VEC) {
        p = load<8>(xr + (c < cols ? c : 0));
        if (c >= cols) p = Pack<T, 8>{};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const T t = xr[min(c + i, cols - 1)];
            p.v[i] = c + i < cols ? t : T{};
        }
    }
    return p;
}

struct AdapterArgs {
    const void *x;
    const int32_t *slot;
    const float *base;
    float *y;
    const char *data;
    const AdapterMeta *meta;
    int64_t ldx, ldbase, ldy;
    size_t slot_bytes;
    int M, slots, rows, cols, rank_tiles, col_blocks, row_tiles;   // of the resident layout: 16 ranks, 32 columns, 16 rows
    int splits;      // workgroups that share the outputs of a row, or of a tile of rows
    bool vec_y;      // base and y rows start at 16 bytes and have a multiple of four columns
};

EIF_DEV int slot_of(const AdapterArgs &a, int row)
{
    const int s = a.slot[row];
    return (unsigned)s < (unsigned)a.slots ? s : -1;
}

// f with the count of 16-rank tiles that are taken at a time: 1, 2 or 4 (of 3: the fourth is computed of what lies there and not used).
template <typename F>
EIF_DEV void by_tiles(int n, F f)
{
    if (n == 1) f(std::integral_constant<int, 1>{});
    else if (n == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 4>{});
}

// A few rows: a workgroup of 16 waves has one row and 1024 of its outputs. It computes the row's whole A x, which workgroups of the
// same row repeat (out of the XCD's L2, where they all run), and from it its outputs: one launch instead of two with the sums of the
// first in memory between them.
template <typename X, typename W, bool VEC>
__global__ __launch_bounds__(1024) void adapter_rows_kernel(AdapterArgs a)
{
    __shared__ float part[16][kMaxRank];
    __shared__ v4f v[kMaxRank / 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t16 = lane & 15, q = lane >> 4;
    const int i8 = blockIdx.x / 8, row = i8 / a.splits * 8 + blockIdx.x % 8, n0 = i8 % a.splits * 1024;
    if (row >= a.M) return;
    const int s = slot_of(a, row), n = n0 + tid;
    const float base = a.base && n < a.rows ? a.base[row * a.ldbase + n] : 0.0f;
    float *y = a.y + row * a.ldy + n;
    const int rank = s < 0 ? 0 : a.meta[s].rank;
    if (rank == 0) {
        if (n < a.rows) *y = base;
        return;
    }
    const X *x = static_cast<const X *>(a.x) + row * a.ldx;
    const W *A = reinterpret_cast<const W *>(a.data + s * a.slot_bytes);
    const W *B = A + (size_t)a.rank_tiles * a.col_blocks * 512;
    const int tiles = (rank + 15) / 16;
    for (int r0 = 0; r0 < tiles; r0 += 4) {
        by_tiles(min(tiles - r0, 4), [&](auto n_) {
            constexpr int RN = decltype(n_)::value, U = RN == 4 ? 2 : 4;
            float acc[RN] = {};
            for (int cb = wave; cb < a.col_blocks; cb += 16 * U) {
                Pack<W, 8> w[U][RN];
                Pack<X, 8> xv[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int b = min(cb + 16 * u, a.col_blocks - 1);
                    xv[u] = x_pack<VEC>(x, b * 32 + q * 8, a.cols);
#pragma unroll
                    for (int r = 0; r < RN; ++r)
                        w[u][r] = load<8>(A + ((size_t)min(r0 + r, a.rank_tiles - 1) * a.col_blocks + b) * 512 + lane * 8);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (cb + 16 * u >= a.col_blocks) break;
#pragma unroll
                    for (int r = 0; r < RN; ++r) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) acc[r] = fmaf(to_f32(xv[u].v[j]), to_f32(w[u][r].v[j]), acc[r]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < RN; ++r) {
                acc[r] += xlane<16>(acc[r]);
                acc[r] += xlane<32>(acc[r]);
                if (q == 0 && r0 + r < tiles) part[wave][(r0 + r) * 16 + t16] = acc[r];
            }
        });
    }
    __syncthreads();
    if (tid < tiles * 16) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; ++w) sum += part[w][tid];
        reinterpret_cast<float *>(v)[tid] = tid < rank ? sum * a.meta[s].scale : 0.0f;   // an infinite x makes NaN of the zeros beyond the rank
    }
    __syncthreads();
    // a wave has 4 tiles of 16 outputs; a lane sums its ranks, and the four lanes of an output meet in the lane whose output it is
    const int nt0 = n0 / 16 + wave * 4;
    if (nt0 >= a.row_tiles) return;
    float sum[4] = {};
    for (int r = 0; r < tiles; ++r) {
        const v4f vr = v[r * 4 + q];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const Pack<W, 4> w = load<4>(B + ((size_t)min(nt0 + t, a.row_tiles - 1) * 64 + lane) * a.rank_tiles * 4 + r * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[t] = fmaf(to_f32(w.v[j]), vr[j], sum[t]);
        }
    }
    const bool high = lane & 32, odd = lane & 16;
    const float k0 = (high ? sum[2] : sum[0]) + xlane<32>(high ? sum[0] : sum[2]);
    const float k1 = (high ? sum[3] : sum[1]) + xlane<32>(high ? sum[1] : sum[3]);
    const float out = (odd ? k1 : k0) + xlane<16>(odd ? k0 : k1);
    if (n < a.rows) *y = base + out;
}

// W x, 16 ranks by 16 tokens by 32 columns, on a lane's 8 columns of each. Of one 16-bit type: one instruction, whose products are
// exact; else as FP32, four columns at a time.
template <typename X, typename W>
EIF_DEV v4f product32(const Pack<W, 8> &w, const Pack<X, 8> &x, v4f acc)
{
    if constexpr (std::is_same<X, W>::value && std::is_same<X, __hip_bfloat16>::value) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), acc, 0, 0, 0);
    } else if constexpr (std::is_same<X, W>::value && std::is_same<X, __half>::value) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, x), acc, 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w.v[j]), to_f32(x.v[j]), acc, 0, 0, 0);
        return acc;
    }
}

// A float as the sum of three bf16, exactly (8 bits of its 24 each), four at a time; an infinity or NaN is in the first alone.
EIF_DEV void planes4(v4f v, uint2 *p)
{
    uint32_t h[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[0][j] = __float_as_uint(v[j]) & 0xffff0000u;
        const float first = __uint_as_float(h[0][j]), rest = v[j] == first ? 0.0f : v[j] - first;
        h[1][j] = __float_as_uint(rest) & 0xffff0000u;
        h[2][j] = __float_as_uint(rest - __uint_as_float(h[1][j]));
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        p[i] = make_uint2(__builtin_amdgcn_perm(h[i][1], h[i][0], 0x07060302), __builtin_amdgcn_perm(h[i][3], h[i][2], 0x07060302));
}

// Many rows: a workgroup of 8 waves has 16 rows and a share of their outputs, and takes the adapters that its rows name one after
// another (rows of a prompt share theirs). First V = A x of the 16 rows: the waves split the columns, and their sums meet in LDS. Then
// B V, a tile of 16 outputs at a time, the tokens being the columns in both products. bf16 B: V as three bf16 planes on 16x16x32
// instructions, whose products are exact, a sixteenth of the time of FP32 ones; else FP32 instructions.
template <typename X, typename W, bool VEC>
__global__ __launch_bounds__(512) void adapter_tile_kernel(AdapterArgs a)
{
    constexpr bool planes = std::is_same<W, __hip_bfloat16>::value;
    __shared__ v4f part[8][4][64];
    __shared__ v4f vs[planes ? 1 : kMaxRank / 16][64];                       // V [16 ranks][lane]
    __shared__ uint4 vp[planes ? kMaxRank / 32 : 1][3][64];                  // [32 ranks][plane][lane]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t16 = lane & 15, q = lane >> 4;
    const int i8 = blockIdx.x / 8, tile = i8 / a.splits * 8 + blockIdx.x % 8, split = i8 % a.splits;
    if (tile * 16 >= a.M) return;
    const int row = min(tile * 16 + t16, a.M - 1);
    int s = slot_of(a, row);
    if (s >= 0 && a.meta[s].rank == 0) s = -1;
    const bool live = tile * 16 + t16 < a.M;
    const X *x = static_cast<const X *>(a.x) + row * a.ldx;
    const float *base = a.base ? a.base + row * a.ldbase : nullptr;
    float *y = a.y + row * a.ldy;
    const int groups = (a.row_tiles + 3) / 4;   // of four tiles of outputs
    const int from = (int)((int64_t)groups * split / a.splits), to = (int)((int64_t)groups * (split + 1) / a.splits);

    // the same in every wave: which of the 16 rows are left
    uint32_t left = (uint32_t)__ballot(live) & 0xffff;
    while (left) {
        const int now = __builtin_amdgcn_readlane(s, __builtin_ctz(left));
        const bool mine = live && s == now;
        left &= ~(uint32_t)__ballot(mine);
        if (now < 0 && a.base == a.y) continue;
        const int rank = now < 0 ? 0 : a.meta[now].rank, tiles = (rank + 15) / 16;
        const W *A = reinterpret_cast<const W *>(a.data + max(now, 0) * a.slot_bytes);
        const W *B = A + (size_t)a.rank_tiles * a.col_blocks * 512;
        const float scale = now < 0 ? 0.0f : a.meta[now].scale;
        for (int r0 = 0; r0 < tiles; r0 += 4) {
            const int rn = min(tiles - r0, 4);
            by_tiles(rn, [&](auto n_) {
                constexpr int RN = decltype(n_)::value, U = RN == 4 ? 2 : 4;
                v4f acc[RN] = {};
                for (int cb = wave * U; cb < a.col_blocks; cb += 8 * U) {
                    Pack<W, 8> w[U][RN];
                    Pack<X, 8> xv[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int b = min(cb + u, a.col_blocks - 1);
                        xv[u] = x_pack<VEC>(x, b * 32 + q * 8, a.cols);
#pragma unroll
                        for (int r = 0; r < RN; ++r)
                            w[u][r] = load<8>(A + ((size_t)min(r0 + r, a.rank_tiles - 1) * a.col_blocks + b) * 512 + lane * 8);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (cb + u >= a.col_blocks) break;
#pragma unroll
                        for (int r = 0; r < RN; ++r) acc[r] = product32(w[u][r], xv[u], acc[r]);
                    }
                }
#pragma unroll
                for (int r = 0; r < RN; ++r) part[wave][r][lane] = acc[r];
            });
            __syncthreads();
            if (wave < 4) {
                v4f sum = {};
                if (wave < rn) {
#pragma unroll
                    for (int w = 0; w < 8; ++w) sum += part[w][wave][lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[j] = (r0 + wave) * 16 + q * 4 + j < rank ? sum[j] * scale : 0.0f;
                }
                if constexpr (planes) {
                    uint2 p[3];
                    planes4(sum, p);
#pragma unroll
                    for (int i = 0; i < 3; ++i) reinterpret_cast<uint2 *>(&vp[(r0 + wave) / 2][i][lane])[wave & 1] = p[i];
                } else {
                    vs[r0 + wave][lane] = sum;
                }
            }
            __syncthreads();
        }
        const int pairs = (tiles + 1) / 2;
        for (int g = from + wave; g < to; g += 8) {
            const int nt0 = g * 4, n0 = nt0 * 16 + q * 4;
            v4f add[4], acc[4] = {};
            const W *Bl[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int n = n0 + t * 16;
                add[t] = v4f{};
                if (mine && base) {
                    if (a.vec_y) {
                        if (n < a.rows) add[t] = *reinterpret_cast<const v4f *>(base + n);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (n + j < a.rows) add[t][j] = base[n + j];
                    }
                }
                Bl[t] = B + ((size_t)min(nt0 + t, a.row_tiles - 1) * 64 + lane) * a.rank_tiles * 4;
            }
            if constexpr (planes) {
                for (int p = 0; p < pairs; ++p) {
                    uint4 w[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint2 *b = reinterpret_cast<const uint2 *>(Bl[t] + p * 8);
                        const uint2 lo = b[0], hi = p * 2 + 1 < tiles ? b[1] : make_uint2(0, 0);
                        w[t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                    }
#pragma unroll
                    for (int i = 2; i >= 0; --i) {
                        const uint4 v = vp[p][i][lane];
#pragma unroll
                        for (int t = 0; t < 4; ++t)
                            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[t]), __builtin_bit_cast(v8bf, v), acc[t], 0, 0, 0);
                    }
                }
            } else {
                for (int r = 0; r < tiles; ++r) {
                    const v4f v = vs[r][lane];
                    Pack<W, 4> w[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) w[t] = load<4>(Bl[t] + r * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w[t].v[j]), v[j], acc[t], 0, 0, 0);
                    }
                }
            }
            if (!mine) continue;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int n = n0 + t * 16;
                const v4f o = add[t] + acc[t];
                if (a.vec_y) {
                    if (n < a.rows) *reinterpret_cast<v4f *>(y + n) = o;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (n + j < a.rows) y[n + j] = o[j];
                }
            }
        }
        __syncthreads();   // V is the next adapter's
    }
}

// An adapter into its place, zeros around it, and its rank and scale.
template <typename W>
__global__ __launch_bounds__(256) void adapter_set_kernel(const W *A, int64_t lda, const W *B, int64_t ldb, int rank, float scale, int rows,
                                                          int cols, int rank_tiles, int col_blocks, int row_tiles, W *to, AdapterMeta *meta)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, na = (int64_t)rank_tiles * col_blocks * 512, nb = (int64_t)row_tiles * rank_tiles * 256;
    if (i == 0) *meta = {rank, scale};
    if (i >= na + nb) return;
    W v{};
    if (i < na) {
        const int lane = (int)(i / 8) & 63, r = (int)(i / 512 / col_blocks) * 16 + lane % 16, c = (int)(i / 512 % col_blocks) * 32 + lane / 16 * 8 + (int)(i & 7);
        if (r < rank && c < cols) v = A[r * lda + c];
    } else {
        const int64_t k = i - na, of_lane = k / (rank_tiles * 4);
        const int at = (int)(k - of_lane * (rank_tiles * 4)), lane = (int)of_lane & 63;
        const int n = (int)(of_lane / 64) * 16 + lane % 16, r = at / 4 * 16 + lane / 16 * 4 + at % 4;
        if (n < rows && r < rank) v = B[n * ldb + r];
    }
    to[i] = v;
}

// ---- launches ----

template <typename X, typename W>
int launch_adapters_as(AdapterArgs a, hipStream_t st)
{
    const bool vec = aligned(a.x, 16) && a.ldx % 8 == 0 && a.cols % 8 == 0;
    if (a.M <= 64) {
        a.splits = eif_ceil_div(a.rows, 1024);
        const unsigned blocks = (unsigned)(eif_ceil_div(a.M, 8) * 8 * a.splits);
        if (vec)
            adapter_rows_kernel<X, W, true><<<blocks, 1024, 0, st>>>(a);
        else
            adapter_rows_kernel<X, W, false><<<blocks, 1024, 0, st>>>(a);
    } else {
        const int tiles = eif_ceil_div(a.M, 16);
        a.splits = std::max(1, std::min(eif_ceil_div(a.rows, 128), 512 / tiles));
        const unsigned blocks = (unsigned)(eif_ceil_div(tiles, 8) * 8 * a.splits);
        if (vec)
            adapter_tile_kernel<X, W, true><<<blocks, 512, 0, st>>>(a);
        else
            adapter_tile_kernel<X, W, false><<<blocks, 512, 0, st>>>(a);
    }
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

template <typename X>
int launch_adapters(const AdapterArgs &a, int type, hipStream_t st)
{
    if (type == EIF_HIP_F32) return launch_adapters_as<X, float>(a, st);
    return type == EIF_HIP_F16 ? launch_adapters_as<X, __half>(a, st) : launch_adapters_as<X, __hip_bfloat16>(a, st);
}

template <typename W>
int launch_set(const eif_hip_adapters *h, int slot, int rank, const void *A, int64_t lda, const void *B, int64_t ldb, float scale,
               hipStream_t st)
{
    const int64_t n = (int64_t)h->rank_pad * (h->cols_pad + h->rows_pad);
    adapter_set_kernel<W><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
        static_cast<const W *>(A), lda, static_cast<const W *>(B), ldb, rank, scale, h->rows, h->cols, h->rank_pad / 16, h->cols_pad / 32,
        h->rows_pad / 16,        reinterpret_cast<W *>(h->data + slot * h->slot_bytes), h->meta + slot);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

int check_device(const eif_hip_adapters *a)
{
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess) return EIF_HIP_E_DEVICE;
    return dev == a->device ? EIF_HIP_OK : EIF_HIP_E_ARG;
}

}  // namespace

extern "C" {

int eif_hip_adapters_create(eif_hip_adapters **out, int slots, int rows, int cols, int max_rank, int type)
{
    if (!out) return EIF_HIP_E_ARG;
    *out = nullptr;
    if (slots < 1 || rows < 1 || cols < 1 || max_rank < 1 || type < EIF_HIP_F32 || type > EIF_HIP_BF16) return EIF_HIP_E_ARG;
    if (slots > kMaxSlots || rows > kMaxDim || cols > kMaxDim || max_rank > kMaxRank) return EIF_HIP_E_LIMIT;
    eif_hip_adapters q{};
    if (hipGetDevice(&q.device) != hipSuccess) return EIF_HIP_E_DEVICE;
    q.slots = slots, q.rows = rows, q.cols = cols, q.max_rank = max_rank, q.type = type;
    q.rank_pad = eif_round_up(max_rank, kRankPad), q.cols_pad = eif_round_up(cols, kColsPad), q.rows_pad = eif_round_up(rows, kRowsPad);
    q.slot_bytes = (size_t)q.rank_pad * (q.cols_pad + q.rows_pad) * type_size(type);
    const size_t data = slots * q.slot_bytes;
    q.bytes = data + slots * sizeof(AdapterMeta);
    if (hipMalloc(&q.data, q.bytes) != hipSuccess) {
        (void)hipGetLastError();
        return EIF_HIP_E_NOMEM;
    }
    q.meta = reinterpret_cast<AdapterMeta *>(q.data + data);
    int rc = EIF_HIP_OK;
    if (hipMemsetAsync(q.meta, 0, slots * sizeof(AdapterMeta), nullptr) != hipSuccess || hipStreamSynchronize(nullptr) != hipSuccess)
        rc = EIF_HIP_E_DEVICE;
    eif_hip_adapters *h = rc == EIF_HIP_OK ? new (std::nothrow) eif_hip_adapters(q) : nullptr;
    if (!h) {
        (void)hipFree(q.data);
        return rc == EIF_HIP_OK ? EIF_HIP_E_NOMEM : rc;
    }
    *out = h;
    return EIF_HIP_OK;
}

void eif_hip_adapters_destroy(eif_hip_adapters *a)
{
    if (!a) return;
    (void)hipFree(a->data);
    delete a;
}

int eif_hip_adapters_set(eif_hip_adapters *a, int slot, int rank, const void *A, int64_t lda, const void *B, int64_t ldb, float scale,
                         int src_on_device, void *stream)
{
    if (!a || slot < 0 || slot >= a->slots || rank < 0 || rank > a->max_rank) return EIF_HIP_E_ARG;
    const size_t size = type_size(a->type);
    if (rank > 0 && (!A || !B || lda < a->cols || ldb < rank || !std::isfinite(scale) || !aligned(A, size) || !aligned(B, size)))
        return EIF_HIP_E_ARG;
    int rc = check_device(a);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (lda > INT64_MAX / 8 / kMaxRank || ldb > INT64_MAX / 8 / kMaxDim) return EIF_HIP_E_LIMIT;
    char *up = nullptr;
    if (rank > 0 && !src_on_device) {
        const size_t na = ((size_t)(rank - 1) * lda + a->cols) * size, nb = ((size_t)(a->rows - 1) * ldb + rank) * size;
        if (hipMalloc(&up, na + nb) != hipSuccess) {
            (void)hipGetLastError();
            return EIF_HIP_E_NOMEM;
        }
        if (hipMemcpyAsync(up, A, na, hipMemcpyHostToDevice, st) != hipSuccess ||
            hipMemcpyAsync(up + na, B, nb, hipMemcpyHostToDevice, st) != hipSuccess)
            rc = EIF_HIP_E_DEVICE;
        A = up, B = up + na;
    }
    if (rc == EIF_HIP_OK) {
        if (a->type == EIF_HIP_F32)
            rc = launch_set<float>(a, slot, rank, A, lda, B, ldb, scale, st);
        else   // copied as they are, whichever of the two
            rc = launch_set<uint16_t>(a, slot, rank, A, lda, B, ldb, scale, st);
    }
    if (hipStreamSynchronize(st) != hipSuccess && rc == EIF_HIP_OK) rc = EIF_HIP_E_DEVICE;
    if (up) (void)hipFree(up);
    return rc;
}

int eif_hip_adapters_info(const eif_hip_adapters *a, int *slots, int *rows, int *cols, int *max_rank, int *type, size_t *bytes)
{
    if (!a) return EIF_HIP_E_ARG;
    if (slots) *slots = a->slots;
    if (rows) *rows = a->rows;
    if (cols) *cols = a->cols;
    if (max_rank) *max_rank = a->max_rank;
    if (type) *type = a->type;
    if (bytes) *bytes = a->bytes;
    return EIF_HIP_OK;
}

int eif_hip_adapters_linear(const eif_hip_adapters *h, const void *x, int type, int64_t ldx, const int32_t *slot, const float *base,
                            int64_t ldbase, float *y, int64_t ldy, int M, void *stream)
{
    if (!h || M < 0 || type < EIF_HIP_F32 || type > EIF_HIP_BF16) return EIF_HIP_E_ARG;
    if (ldx < h->cols || ldy < h->rows || (base && ldbase < h->rows) || (base == y && ldbase != ldy)) return EIF_HIP_E_ARG;
    if (M > kMaxM) return EIF_HIP_E_LIMIT;
    int rc = check_device(h);
    if (rc || M == 0) return rc;
    if (!x || !slot || !y || !aligned(x, type_size(type)) || !aligned(slot, 4) || !aligned(base, 4) || !aligned(y, 4)) return EIF_HIP_E_ARG;
    AdapterArgs a{};
    a.x = x, a.slot = slot, a.base = base, a.y = y, a.data = h->data, a.meta = h->meta, a.ldx = ldx, a.ldbase = ldbase, a.ldy = ldy;
    a.slot_bytes = h->slot_bytes, a.M = M, a.slots = h->slots, a.rows = h->rows, a.cols = h->cols;
    a.rank_tiles = h->rank_pad / 16, a.col_blocks = h->cols_pad / 32, a.row_tiles = h->rows_pad / 16;
    a.vec_y = aligned(y, 16) && ldy % 4 == 0 && h->rows % 4 == 0 && (!base || (aligned(base, 16) && ldbase % 4 == 0));
    hipStream_t st = (hipStream_t)stream;
    if (type == EIF_HIP_F32) return launch_adapters<float>(a, h->type, st);
    return type == EIF_HIP_F16 ? launch_adapters<__half>(a, h->type, st) : launch_adapters<__hip_bfloat16>(a, h->type, st);
}

}  // extern "C"
