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
//   B [16 rows][32 ranks][lane][8]: lane l has row l % 16 of the 16 and ranks 4 (l / 16) .. + 3 of the first 16, then of the other 16;
//     where the last 32 are only 16, [lane][4].
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

// Where a lane's part of 16 rows' B begins, and in it that of ranks 16 r .. + 15.
EIF_DEV int b_part(int r, int rank_tiles, int lane) { return (r >> 1) * 512 + (r + 1 == rank_tiles && !(r & 1) ? lane * 4 : lane * 8 + (r & 1) * 4); }

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
    int tiles_xcd;   // tiles of rows that an XCD takes, one behind the other: rows of a prompt share an adapter, and its L2 holds it
    bool vec_y;      // base and y rows start at 16 bytes and have a multiple of four columns
};

EIF_DEV int slot_of(const AdapterArgs &a, int row)
{
    const int s = a.slot[row];
    return (unsigned)s < (unsigned)a.slots ? s : -1;
}

// f with the count of 16-rank tiles that are taken at a time: 1, 2 or 4 (of 3, the fourth is computed of what lies there and not used).
template <typename F>
EIF_DEV void by_tiles(int n, F f)
{
    if (n == 1) f(std::integral_constant<int, 1>{});
    else if (n == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 4>{});
}

// A few rows: a workgroup of 16 waves has one row and 1024 of its outputs. It computes the row's whole A x, which workgroups of the
// same row repeat (out of the XCD's L2, where they all run), and from it its outputs: one launch instead of two with the sums of the
// first in memory between them. x, which 16 lanes share, comes from LDS, so as not to pass the L1 16 times over. ONE: ranks up to 16, whose
// matrices are read before the rank is known (what lies behind it is zeros).
// Bound by one workgroup's chain (slot, rank, x, A, the waves' sums, B), which grows with the ranks. One row of 16 ranks through
// 2560x2560 3.8 us, of which 1.7 are an empty launch's. 48 rows through 4096x4096: 5.7 us with 16 ranks, 9.2 with 32, 13.4 with 64;
// of the last, 10.5 remain with 8 rows in place of 48, 10.7 with 64 columns in place of 4096, 11.9 with 16 outputs. 48 rows of 48
// requests with 8 to 64 ranks 11.4.
template <typename X, typename W, bool VEC, bool ONE>
__global__ __launch_bounds__(1024) void adapter_rows_kernel(AdapterArgs a)
{
    constexpr int R = ONE ? 16 : kMaxRank, kCols = 4096;
    __shared__ float part[16][R];
    __shared__ v4f v[R / 4];
    __shared__ v4f xs[kCols / 4];   // columns of x
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t16 = lane & 15, q = lane >> 4;
    const int i8 = blockIdx.x / 8, row = i8 / a.splits * 8 + blockIdx.x % 8, n0 = i8 % a.splits * 1024;
    if (row >= a.M) return;
    const X *x = static_cast<const X *>(a.x) + row * a.ldx;
    const auto x_quad = [&](int c) {   // four columns, zeros behind the last
        v4f r = {};
        if constexpr (VEC) {
            if (c < a.cols) {
                const Pack<X, 4> p = load<4>(x + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = to_f32(p.v[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < a.cols) r[j] = to_f32(x[c + j]);
        }
        return r;
    };
    const v4f x0 = x_quad(tid * 4);
    const int s = slot_of(a, row), n = n0 + tid;
    const float base = a.base && n < a.rows ? a.base[row * a.ldbase + n] : 0.0f;
    float *y = a.y + row * a.ldy + n;
    const AdapterMeta meta = s < 0 ? AdapterMeta{} : a.meta[s];
    if (ONE ? s < 0 : meta.rank == 0) {
        if (n < a.rows) *y = base;
        return;
    }
    const W *A = reinterpret_cast<const W *>(a.data + s * a.slot_bytes);
    const W *B = A + (size_t)a.rank_tiles * a.col_blocks * 512;
    const int tiles = ONE ? 1 : (meta.rank + 15) / 16;
    for (int r0 = 0; r0 < tiles; r0 += 4) {
        by_tiles(ONE ? 1 : min(tiles - r0, 4), [&](auto n_) {
            constexpr int RN = decltype(n_)::value, U = (RN == 4 ? 4 : 8) / (sizeof(W) == 4 ? 2 : 1);
            float acc[RN] = {};
            for (int k = 0; k < a.col_blocks; k += kCols / 32) {   // a wave has every 16th block of 32 columns
                const int end = min(k + kCols / 32, a.col_blocks);
                for (int cb = k + wave; cb < k + kCols / 32; cb += 16 * U) {
                    Pack<W, 8> w[U][RN];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
#pragma unroll
                        for (int r = 0; r < RN; ++r)
                            w[u][r] = load<8>(A + ((size_t)min(r0 + r, a.rank_tiles - 1) * a.col_blocks + min(cb + 16 * u, end - 1)) * 512 + lane * 8);
                    }
                    if (cb == k + wave && (r0 == 0 || a.col_blocks > kCols / 32)) {   // the waves' loads are under way
                        if (r0 + k > 0) __syncthreads();
                        xs[tid] = k == 0 && r0 == 0 ? x0 : x_quad(k * 32 + tid * 4);
                        __syncthreads();
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (cb + 16 * u < end) {
                            const v4f lo = xs[(cb + 16 * u - k) * 8 + q * 2], hi = xs[(cb + 16 * u - k) * 8 + q * 2 + 1];
#pragma unroll
                            for (int r = 0; r < RN; ++r) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) acc[r] = fmaf(j < 4 ? lo[j & 3] : hi[j & 3], to_f32(w[u][r].v[j]), acc[r]);
                            }
                        }
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
    // a wave has 4 tiles of 16 outputs; B's first ranks are on their way while the waves' sums meet
    constexpr int RB = ONE ? 1 : 4;
    const int nt0 = n0 / 16 + wave * 4;
    Pack<W, 4> bw[4][RB];
    const W *Bt[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        Bt[t] = B + (size_t)min(nt0 + t, a.row_tiles - 1) * a.rank_tiles * 256;
#pragma unroll
        for (int r = 0; r < RB; ++r) bw[t][r] = load<4>(Bt[t] + b_part(min(r, tiles - 1), a.rank_tiles, lane));
    }
    __syncthreads();
    if (tid < tiles * 16) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; ++w) sum += part[w][tid];
        reinterpret_cast<float *>(v)[tid] = tid < meta.rank ? sum * meta.scale : 0.0f;   // an infinite x makes NaN of the zeros beyond the rank
    }
    __syncthreads();
    if (nt0 >= a.row_tiles) return;
    if (ONE && meta.rank == 0) {   // what an empty slot holds is nothing to compute with
        if (n < a.rows) *y = base;
        return;
    }
    // a lane sums its ranks, and the four lanes of an output meet in the lane whose output it is
    float sum[4] = {};
    for (int r0 = 0; r0 < tiles; r0 += RB) {
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            if (r0 + r >= tiles) break;
            const v4f vr = v[(r0 + r) * 4 + q];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[t] = fmaf(to_f32(bw[t][r].v[j]), vr[j], sum[t]);
            }
        }
        if (r0 + RB < tiles) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int r = 0; r < RB; ++r) bw[t][r] = load<4>(Bt[t] + b_part(min(r0 + RB + r, tiles - 1), a.rank_tiles, lane));
            }
        }
    }
    const bool high = lane & 32, odd = lane & 16;
    const float k0 = (high ? sum[2] : sum[0]) + xlane<32>(high ? sum[0] : sum[2]);
    const float k1 = (high ? sum[3] : sum[1]) + xlane<32>(high ? sum[1] : sum[3]);
    const float out = (odd ? k1 : k0) + xlane<16>(odd ? k0 : k1);
    if (n < a.rows) *y = base + out;
}

// A float as the sum of three bf16, exactly (8 bits of its 24 each) down to bf16's least number, 2^-133, four at a time; an infinity or
// NaN is in the first alone. The others may be 0, which an infinite factor makes NaN.
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

// Many rows: a workgroup of 8 waves has TT tiles of 16 rows and a share of their outputs. First V = A x of the rows, for all the
// adapters that they name (rows of a prompt share theirs), 4 tiles of 16 ranks at a time: the waves split the columns, and their
// sums meet in LDS, where each row keeps those of its own adapter. Then base + B V, two tiles of 16 outputs at a time, with every adapter in
// turn, each row taking its own one's. The tokens are the columns of both products. bf16 B: V as three bf16 planes on 16x16x32
// instructions, whose products are exact, a sixteenth of the time of FP32 ones; else FP32 instructions. Loads run ahead: x and A two or
// four steps, base and B two or three. 8192 bf16 rows of 64 ranks through 4096x4096 87 us where they share an adapter (3.9 TB/s: 25 us the
// first product with its launch, 66 the second, copying base to y 58), 113 where nine requests meet in tiles, whose workgroups go
// through x and the outputs for two adapters and end last; 116 with f16 matrices. 1531 FP32 rows of 16 ranks through 6912x2560 31 us (3.2
// TB/s), 28 where they share an adapter.
template <typename X, typename W, bool VEC, int TT>
__global__ __launch_bounds__(512, TT == 1 ? 4 : 2) void adapter_tile_kernel(AdapterArgs a)
{
    constexpr bool planes = std::is_same<W, __hip_bfloat16>::value;
    constexpr int kChunk = 4;   // tiles of 16 ranks that a pass over x takes, and a step of the second product
    constexpr int DX = !VEC ? 1 : sizeof(X) == 2 && planes ? 4 : 2;   // steps of x under way, as many as the registers hold
    constexpr int DW = VEC && sizeof(W) == 2 ? 2 : 1;                 // and of A; DX is a multiple of it
    __shared__ v4f part[8][kChunk][TT][64];
    __shared__ v4f vs[planes ? 1 : kMaxRank / 16][TT][64];          // V [16 ranks][tile of rows][lane]
    __shared__ uint4 vp[planes ? kMaxRank / 32 : 1][3][TT][64];     // [32 ranks][plane][tile of rows][lane]
    __shared__ int2 tile_at[TT * 16 * kMaxRank / 16];               // what the first product goes through: slot, tile of ranks
    __shared__ int2 step_at[TT * 16 * kMaxRank / 16 / kChunk];      // and the second: slot, first tile of ranks
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t16 = lane & 15, q = lane >> 4;
    const int i8 = blockIdx.x / 8, tile = (int)(blockIdx.x % 8) * a.tiles_xcd + i8 / a.splits, split = i8 % a.splits;
    if (i8 / a.splits >= a.tiles_xcd || tile * (16 * TT) >= a.M) return;
    int row[TT], s[TT];
    bool live[TT];
    const X *x[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const int r = (tile * TT + t) * 16 + t16;
        live[t] = r < a.M;
        row[t] = min(r, a.M - 1);
        x[t] = static_cast<const X *>(a.x) + row[t] * a.ldx;
    }
    const int per = (a.col_blocks + 7) / 8, c0 = wave * per, c1 = min(c0 + per, a.col_blocks);
    Pack<X, 8> xr[DX][TT];
    const auto load_x = [&](Pack<X, 8> *p, int b) {
#pragma unroll
        for (int t = 0; t < TT; ++t) p[t] = x_pack<VEC>(x[t], min(b, a.col_blocks - 1) * 32 + q * 8, a.cols);
    };
#pragma unroll
    for (int u = 0; u < DX; ++u) load_x(xr[u], c0 + u);
    uint32_t left = 0;   // rows whose adapter is still to come
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        s[t] = slot_of(a, row[t]);
        if (s[t] >= 0 && a.meta[s[t]].rank == 0) s[t] = -1;
        left |= ((uint32_t)__ballot(live[t] && s[t] >= 0) & 0xffff) << (16 * t);
    }

    int all = 0, steps = 0, most = 0;   // tiles of ranks, steps of the second product, the most tiles in one; the same in every wave
    while (left) {
        const int first = __builtin_ctz(left);
        int now = __builtin_amdgcn_readlane(s[0], first & 15);
        if (TT == 2 && first >= 16) now = __builtin_amdgcn_readlane(s[TT - 1], first & 15);
#pragma unroll
        for (int t = 0; t < TT; ++t) left &= ~(((uint32_t)__ballot(s[t] == now) & 0xffff) << (16 * t));
        const int tiles = (a.meta[now].rank + 15) / 16;
        for (int r = 0; r < tiles; r += kChunk, ++steps) {
            if (tid < min(tiles - r, kChunk)) tile_at[all + r + tid] = make_int2(now, r + tid);
            if (tid == 0) step_at[steps] = make_int2(now, r);
        }
        all += tiles;
        most = max(most, min(tiles, kChunk));
    }
    __syncthreads();
    for (int e0 = 0; e0 < all; e0 += kChunk) {
        if (e0 > 0) {
#pragma unroll
            for (int u = 0; u < DX; ++u) load_x(xr[u], c0 + u);
        }
        by_tiles(min(all - e0, kChunk), [&](auto n_) {
            constexpr int RN = decltype(n_)::value;
            const W *Ar[RN];
#pragma unroll
            for (int r = 0; r < RN; ++r) {
                const int2 e = tile_at[min(e0 + r, all - 1)];
                const int slot = __builtin_amdgcn_readfirstlane(e.x), rt = __builtin_amdgcn_readfirstlane(e.y);
                Ar[r] = reinterpret_cast<const W *>(a.data + slot * a.slot_bytes) + (size_t)rt * a.col_blocks * 512;
            }
            v4f acc[RN][TT] = {};
            Pack<W, 8> w[DW][RN];
            const auto load_w = [&](Pack<W, 8> *p, int b) {
#pragma unroll
                for (int r = 0; r < RN; ++r) p[r] = load<8>(Ar[r] + (size_t)min(b, a.col_blocks - 1) * 512 + lane * 8);
            };
#pragma unroll
            for (int u = 0; u < DW; ++u) load_w(w[u], c0 + u);
            for (int cb = c0; cb < c1; cb += DX) {
#pragma unroll
                for (int u = 0; u < DX; ++u) {
                    if (cb + u < c1) {
                        if constexpr (planes && sizeof(X) == 4) {
                            // x as planes too: 1024 rows of 64 ranks 34 us, with FP32 instructions 50; of 16 ranks as long either way
#pragma unroll
                            for (int t = 0; t < TT; ++t) {
                                uint2 lo[3], hi[3];
                                planes4(v4f{xr[u][t].v[0], xr[u][t].v[1], xr[u][t].v[2], xr[u][t].v[3]}, lo);
                                planes4(v4f{xr[u][t].v[4], xr[u][t].v[5], xr[u][t].v[6], xr[u][t].v[7]}, hi);
#pragma unroll
                                for (int i = 2; i >= 0; --i) {
                                    const v8bf p = __builtin_bit_cast(v8bf, make_uint4(lo[i].x, lo[i].y, hi[i].x, hi[i].y));
#pragma unroll
                                    for (int r = 0; r < RN; ++r)
                                        acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w[u % DW][r]), p, acc[r][t], 0, 0, 0);
                                }
                            }
                        } else {
#pragma unroll
                            for (int r = 0; r < RN; ++r) {
#pragma unroll
                                for (int t = 0; t < TT; ++t) acc[r][t] = product32(w[u % DW][r], xr[u][t], acc[r][t]);
                            }
                        }
                        load_x(xr[u], cb + u + DX);
                        load_w(w[u % DW], cb + u + DW);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < RN; ++r) {
#pragma unroll
                for (int t = 0; t < TT; ++t) part[wave][r][t][lane] = acc[r][t];
            }
        });
        __syncthreads();
        const int r = wave / TT, t = wave % TT, e = e0 + r;   // a wave sums a tile of ranks of a tile of rows
        if (r < kChunk && e < all) {
            const int2 at = tile_at[e];
            const int slot = __builtin_amdgcn_readfirstlane(at.x), rt = __builtin_amdgcn_readfirstlane(at.y);
            const AdapterMeta meta = a.meta[slot];
            v4f sum = part[0][r][t][lane];
#pragma unroll
            for (int w = 1; w < 8; ++w) sum += part[w][r][t][lane];
            // an infinite x makes NaN of the zeros beyond the rank
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] = rt * 16 + q * 4 + j < meta.rank ? sum[j] * meta.scale : 0.0f;
            if ((TT == 1 || t == 0 ? s[0] : s[TT - 1]) == slot) {
                const auto put = [&](int i, v4f v) {
                    if constexpr (planes) {
                        uint2 p[3];
                        planes4(v, p);
#pragma unroll
                        for (int k = 0; k < 3; ++k) reinterpret_cast<uint2 *>(&vp[i / 2][k][t][lane])[i & 1] = p[k];
                    } else {
                        vs[i][t][lane] = v;
                    }
                };
                put(rt, sum);
                if ((rt + 1) * 16 >= meta.rank)   // zeros up to the end of the step
                    for (int i = rt + 1; i % kChunk != 0; ++i) put(i, v4f{});
            }
        }
        __syncthreads();
    }

    const bool in_place = a.base == a.y;
    if (steps == 0 && in_place) return;
    const int groups = (a.row_tiles + 1) / 2;   // of two tiles of outputs
    const int from = (int)((int64_t)groups * split / a.splits), to = (int)((int64_t)groups * (split + 1) / a.splits);
    // rows often lie a power of two apart: tiles of rows begin at different outputs, so as not to meet in the same memory channels
    const int turn = to > from ? (int)((unsigned)(tile * TT) * 5u % (unsigned)(to - from)) : 0;
    const auto tile_of = [&](int g) { return 2 * (g + turn < to ? g + turn : g + turn - (to - from)); };
    const auto load_base = [&](int t, int n) {
        v4f v = {};
        if (a.base) {
            const float *base = a.base + row[t] * a.ldbase;
            if (a.vec_y) {
                v = *reinterpret_cast<const v4f *>(base + min(n, a.rows - 4));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = base[min(n + j, a.rows - 1)];
            }
        }
        return v;
    };
    const auto store_y = [&](int t, int n, v4f v) {
        if (!live[t] || (s[t] < 0 && in_place)) return;
        float *y = a.y + row[t] * a.ldy;
        if (a.vec_y) {
            // past the caches with tiles of 16 rows (1531 rows through 6912x2560 31 us, 42 without), not with those of 32 (8192 rows
            // through 4096x4096 92 us, 87 without)
            if (n < a.rows) {
                if constexpr (TT == 1) __builtin_nontemporal_store(v, reinterpret_cast<v4f *>(y + n));
                else *reinterpret_cast<v4f *>(y + n) = v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < a.rows) y[n + j] = v[j];
        }
    };
    if (steps == 0) {
        for (int g = from + wave; g < to; g += 8) {
            const int n = tile_of(g) * 16 + q * 4;
            v4f v[TT][2];
#pragma unroll
            for (int i = 0; i < 2 * TT; ++i) v[i / 2][i % 2] = load_base(i / 2, n + i % 2 * 16);
#pragma unroll
            for (int i = 0; i < 2 * TT; ++i) store_y(i / 2, n + i % 2 * 16, v[i / 2][i % 2]);
        }
        return;
    }
    by_tiles(most, [&](auto n_) {
        constexpr int RT = decltype(n_)::value, D = planes ? 3 : 2;
        struct Ahead {
            v4f add[TT][2];
            Pack<W, 4> w[2][RT];
        } ahead[D];
        int gl = from + wave, sl = 0;   // the group and step to load next
        const auto load_next = [&](Ahead &h) {
            if (gl >= to) return;
            const int nt = tile_of(gl);
            const int2 st = step_at[sl];
            const int slot = __builtin_amdgcn_readfirstlane(st.x), r0 = __builtin_amdgcn_readfirstlane(st.y);
            const W *B = reinterpret_cast<const W *>(a.data + slot * a.slot_bytes) + (size_t)a.rank_tiles * a.col_blocks * 512;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (sl == 0) {
#pragma unroll
                    for (int t = 0; t < TT; ++t) h.add[t][i] = load_base(t, (nt + i) * 16 + q * 4);
                }
                const W *b = B + (size_t)min(nt + i, a.row_tiles - 1) * a.rank_tiles * 256;
                if constexpr (RT == 1) {
                    h.w[i][0] = load<4>(b + b_part(r0, a.rank_tiles, lane));
                } else {
#pragma unroll
                    for (int r = 0; r < RT; r += 2) {
                        if (r0 + r + 1 < a.rank_tiles) {   // both of the 32
                            const Pack<W, 8> p = load<8>(b + (r0 + r) * 256 + lane * 8);
#pragma unroll
                            for (int j = 0; j < 4; ++j) h.w[i][r].v[j] = p.v[j], h.w[i][r + 1].v[j] = p.v[4 + j];
                        } else {
                            h.w[i][r] = h.w[i][r + 1] = load<4>(b + b_part(min(r0 + r, a.rank_tiles - 1), a.rank_tiles, lane));
                        }
                    }
                }
            }
            if (++sl == steps) {
                sl = 0;
                gl += 8;
            }
        };
#pragma unroll
        for (int d = 0; d < D; ++d) load_next(ahead[d]);
        int g = from + wave, at = 0;
        v4f sum[TT][2];
        while (g < to) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (g < to) {
                    Ahead &h = ahead[d];
                    const int2 st = step_at[at];
                    const int r0 = __builtin_amdgcn_readfirstlane(st.y);
                    v4f acc[TT][2] = {};
                    if constexpr (planes) {
#pragma unroll
                        for (int p = 0; p < (RT + 1) / 2; ++p) {
                            v8bf w[2];
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint2 lo = __builtin_bit_cast(uint2, h.w[i][2 * p]);
                                const uint2 hi = RT > 1 ? __builtin_bit_cast(uint2, h.w[i][RT > 1 ? 2 * p + 1 : 0]) : make_uint2(0, 0);
                                w[i] = __builtin_bit_cast(v8bf, make_uint4(lo.x, lo.y, hi.x, hi.y));
                            }
#pragma unroll
                            for (int i = 2; i >= 0; --i) {
#pragma unroll
                                for (int t = 0; t < TT; ++t) {
                                    const v8bf v = __builtin_bit_cast(v8bf, vp[r0 / 2 + p][i][t][lane]);
                                    acc[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[0], v, acc[t][0], 0, 0, 0);
                                    acc[t][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[1], v, acc[t][1], 0, 0, 0);
                                }
                            }
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < RT; ++r) {
#pragma unroll
                            for (int t = 0; t < TT; ++t) {
                                const v4f v = vs[r0 + r][t][lane];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    acc[t][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(h.w[0][r].v[j]), v[j], acc[t][0], 0, 0, 0);
                                    acc[t][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(h.w[1][r].v[j]), v[j], acc[t][1], 0, 0, 0);
                                }
                            }
                        }
                    }
                    const int n = tile_of(g) * 16 + q * 4;
#pragma unroll
                    for (int i = 0; i < 2 * TT; ++i) {
                        v4f &o = sum[i / 2][i % 2];
                        const v4f &p = acc[i / 2][i % 2];
                        if (at == 0) o = h.add[i / 2][i % 2];
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j] = s[i / 2] == st.x ? o[j] + p[j] : o[j];
                        if (at + 1 == steps) store_y(i / 2, n + i % 2 * 16, o);
                    }
                    load_next(h);
                    if (++at == steps) {
                        at = 0;
                        g += 8;
                    }
                }
            }
        }
    });
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
        const int64_t k = i - na, nt = k / (rank_tiles * 256);
        const int at = (int)(k - nt * (rank_tiles * 256)), p = at / 512, in = at % 512;
        const bool half = 2 * p + 1 == rank_tiles;   // 16 ranks alone
        const int lane = half ? in / 4 : in / 8, n = (int)nt * 16 + lane % 16, r = p * 32 + (half ? 0 : in % 8 / 4 * 16) + lane / 16 * 4 + in % 4;
        if (n < rows && r < rank) v = B[n * ldb + r];
    }
    to[i] = v;
}

// ---- launches ----

template <typename X, typename W, bool VEC, int TT>
int launch_tiles_as(AdapterArgs a, int workgroups, hipStream_t st)
{
    const int tiles = eif_ceil_div(a.M, 16 * TT);
    a.tiles_xcd = eif_ceil_div(tiles, 8);
    // workgroups that run at once: one more would begin when the others end (600 rows through 2560x2560 25 us with 600, 19 with 480)
    a.splits = std::max(1, std::min(eif_ceil_div(a.rows, 128), workgroups / (a.tiles_xcd * 8)));
    adapter_tile_kernel<X, W, VEC, TT><<<(unsigned)(a.tiles_xcd * 8 * a.splits), 512, 0, st>>>(a);
    EIF_HIP_LAUNCHED();
    return EIF_HIP_OK;
}

// Tiles of 32 rows read A and B half as often, and leave half as many workgroups, whose stores stay in the caches. us with tiles of 32 / 16:
// 8192 rows of 64 ranks through 4096x4096 87 / 109, with nine requests 113 / 129; 4096 of 64 57 / 67, of 16 50 / 56; 3000 bf16 rows of 64
// ranks 52 / 41, of 16 45 / 32, FP32 rows of 16 51 / 57; 1531 rows of five requests through 6912x2560 42 / 31, 4096 of them 75 / 83.
template <typename X, typename W, bool VEC>
int launch_tiles(const AdapterArgs &a, hipStream_t st)
{
    return a.M >= 4096 ? launch_tiles_as<X, W, VEC, 2>(a, 256, st) : launch_tiles_as<X, W, VEC, 1>(a, 512, st);
}

template <typename X, typename W>
int launch_adapters_as(AdapterArgs a, hipStream_t st)
{
    const bool vec = aligned(a.x, 16) && a.ldx % 8 == 0 && a.cols % 8 == 0;
    // A row a workgroup does not care which adapters meet, a tile does (us, rows of one adapter / of 32 in any order; 512 rows of 16 ranks
    // through 2560x2560: rows 20 / 21, tiles 18 / 79; 256 of 64 through 4096x4096 38 / 49, 30 / 350; 512 72 / 90, 31 / 361; 64 12 / 15, 18 /
    // 200): up to the sizes of a batch of single tokens the rows.
    if (a.M * std::min(a.rank_tiles, 2) <= 512) {
        a.splits = eif_ceil_div(a.rows, 1024);
        const unsigned blocks = (unsigned)(eif_ceil_div(a.M, 8) * 8 * a.splits);
        if (a.rank_tiles == 1)
            vec ? adapter_rows_kernel<X, W, true, true><<<blocks, 1024, 0, st>>>(a) : adapter_rows_kernel<X, W, false, true><<<blocks, 1024, 0, st>>>(a);
        else
            vec ? adapter_rows_kernel<X, W, true, false><<<blocks, 1024, 0, st>>>(a) : adapter_rows_kernel<X, W, false, false><<<blocks, 1024, 0, st>>>(a);
    } else {
        return vec ? launch_tiles<X, W, true>(a, st) : launch_tiles<X, W, false>(a, st);
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
