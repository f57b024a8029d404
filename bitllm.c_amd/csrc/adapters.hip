// adapters.hip -- low-rank adapters of many requests beside a shared projection (eif_hip_adapters.h).
#include "hip_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "../../include/eif_hip_adapters.h"

// Resident: per slot A [rank_pad][cols_pad], then B [rows_pad][rank_pad], of the adapters' type, zeros beyond rank, cols and rows;
// and a rank (0: empty) and scale.
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

// Columns c .. c + N - 1 of a token row, zeros behind the last. VEC: rows start at 16 bytes, their columns are a multiple of eight.
template <int N, bool VEC, typename T>
EIF_DEV void x_values(const T *xr, int c, int cols, float *v)
{
    if constexpr (VEC) {
        const Pack<T, N> p = load<N>(xr + (c < cols ? c : 0));
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = c < cols ? to_f32(p.v[i]) : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = to_f32(xr[min(c + i, cols - 1)]);
            v[i] = c + i < cols ? t : 0.0f;
        }
    }
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
    int M, slots, rows, cols, rank_pad, cols_pad, rows_pad;
    int splits;      // workgroups that share the outputs of a row, or of a tile of rows
    bool vec_y;      // base and y rows start at 16 bytes and have a multiple of four columns
};

EIF_DEV int slot_of(const AdapterArgs &a, int row)
{
    const int s = a.slot[row];
    return (unsigned)s < (unsigned)a.slots ? s : -1;
}

// Sixteen sums over the wave at once: each step hands half of a lane's sums to another lane and takes over half of that one's. A lane
// is left with the sum number index_of_lane(lane).
EIF_DEV float sums16(float *s, int lane)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float give = lane & 1 ? s[i] : s[i + 8], keep = lane & 1 ? s[i + 8] : s[i];
        s[i] = keep + xlane<1>(give);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float give = lane & 2 ? s[i] : s[i + 4], keep = lane & 2 ? s[i + 4] : s[i];
        s[i] = keep + xlane<2>(give);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float give = lane & 4 ? s[i] : s[i + 2], keep = lane & 4 ? s[i + 2] : s[i];
        s[i] = keep + xlane<4>(give);
    }
    const float give = lane & 8 ? s[0] : s[1], keep = lane & 8 ? s[1] : s[0];
    float v = keep + xlane<8>(give);
    v += xlane<16>(v);
    return v + xlane<32>(v);
}
EIF_DEV int index_of_lane(int lane) { return (lane & 1) * 8 + (lane & 2) * 2 + (lane & 4) / 2 + (lane & 8) / 8; }

// A few rows: a workgroup of 16 waves has one row and 1024 of its outputs. It computes the row's whole A x, which workgroups of the
// same row repeat (out of the XCD's L2, where they all run), and from it an output a thread: one launch instead of two with the
// sums of the first in memory between them.
template <typename X, typename W, bool VEC>
__global__ __launch_bounds__(1024) void adapter_rows_kernel(AdapterArgs a)
{
    __shared__ float part[16][kMaxRank];
    __shared__ float v[kMaxRank];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i8 = blockIdx.x / 8, row = i8 / a.splits * 8 + blockIdx.x % 8, n = i8 % a.splits * 1024 + tid;
    if (row >= a.M) return;
    const int s = slot_of(a, row);
    const float base = a.base && n < a.rows ? a.base[row * a.ldbase + n] : 0.0f;
    float *y = a.y + row * a.ldy + n;
    const int rank = s < 0 ? 0 : a.meta[s].rank;
    if (rank == 0) {
        if (n < a.rows) *y = base;
        return;
    }
    const X *x = static_cast<const X *>(a.x) + row * a.ldx;
    const W *A = reinterpret_cast<const W *>(a.data + s * a.slot_bytes);
    const W *B = A + (size_t)a.rank_pad * a.cols_pad;
    for (int r0 = 0; r0 < rank; r0 += 16) {
        float acc[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
        for (int c = tid * 4; c < a.cols_pad; c += 4096) {
            float xv[4];
            x_values<4, VEC>(x, c, a.cols, xv);
            Pack<W, 4> w[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) w[r] = load<4>(A + (size_t)(r0 + r) * a.cols_pad + c);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r] = fmaf(xv[j], to_f32(w[r].v[j]), acc[r]);
            }
        }
        const float sum = sums16(acc, lane);
        if (lane < 16) part[wave][r0 + index_of_lane(lane)] = sum;
    }
    __syncthreads();
    const int ranks = (rank + 15) & ~15;
    if (tid < ranks) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; ++w) sum += part[w][tid];
        v[tid] = tid < rank ? sum * a.meta[s].scale : 0.0f;   // an infinite x makes NaN of the zeros beyond the rank
    }
    __syncthreads();
    if (n >= a.rows) return;
    float out = 0.0f;
    for (int r0 = 0; r0 < ranks; r0 += 16) {
        const Pack<W, 8> lo = load<8>(B + (size_t)n * a.rank_pad + r0), hi = load<8>(B + (size_t)n * a.rank_pad + r0 + 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) out = fmaf(to_f32(lo.v[j]), v[r0 + j], out);
#pragma unroll
        for (int j = 0; j < 8; ++j) out = fmaf(to_f32(hi.v[j]), v[r0 + 8 + j], out);
    }
    *y = base + out;
}

// Many rows: a workgroup of 8 waves has 16 rows and a share of their outputs, and takes the adapters that its rows name one after
// another (rows of a prompt share theirs). First V = A x of the 16 rows: the waves split the columns, and their sums meet in LDS. Then
// B V a tile of 16 outputs at a time. Matrix instructions of FP32 (16x16x4): the tokens are their columns in both products, so that
// a lane's four sums of the first (ranks 4 (lane / 16) .. + 3 of token lane % 16) are its operands of the second.
template <typename X, typename W, bool VEC>
__global__ __launch_bounds__(512) void adapter_tile_kernel(AdapterArgs a)
{
    __shared__ v4f part[8][4][64];
    __shared__ v4f vs[kMaxRank / 16][64];
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
    const int tiles = a.rows_pad / 16, from = (int)((int64_t)tiles * split / a.splits), to = (int)((int64_t)tiles * (split + 1) / a.splits);

    // the same in every wave: which of the 16 rows are left
    uint32_t left = (uint32_t)__ballot(live) & 0xffff;
    while (left) {
        const int now = __builtin_amdgcn_readlane(s, __builtin_ctz(left));
        const bool mine = live && s == now;
        left &= ~(uint32_t)__ballot(mine);
        const int rank = now < 0 ? 0 : a.meta[now].rank, rtiles = (rank + 15) / 16;
        if (now < 0 && a.base == a.y) continue;
        const W *A = reinterpret_cast<const W *>(a.data + max(now, 0) * a.slot_bytes);
        const W *B = A + (size_t)a.rank_pad * a.cols_pad;
        const float scale = now < 0 ? 0.0f : a.meta[now].scale;
        for (int r0 = 0; r0 < rtiles; r0 += 4) {
            const int rn = min(rtiles - r0, 4);
            v4f acc[4] = {};
            for (int c = wave * 32 + q * 8; c < a.cols_pad; c += 256) {
                float xv[8];
                x_values<8, VEC>(x, c, a.cols, xv);
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) {
                    if (rt < rn) {
                        const Pack<W, 8> w = load<8>(A + (size_t)((r0 + rt) * 16 + t16) * a.cols_pad + c);
#pragma unroll
                        for (int j = 0; j < 8; ++j) acc[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w.v[j]), xv[j], acc[rt], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) part[wave][rt][lane] = acc[rt];
            __syncthreads();
            if (wave < rn) {
                v4f sum = part[0][wave][lane];
#pragma unroll
                for (int w = 1; w < 8; ++w) sum += part[w][wave][lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = (r0 + wave) * 16 + q * 4 + j < rank ? sum[j] * scale : 0.0f;
                vs[r0 + wave][lane] = sum;
            }
            __syncthreads();
        }
        for (int nt = from + wave; nt < to; nt += 8) {
            v4f acc = {};
            for (int rt = 0; rt < rtiles; ++rt) {
                const v4f v = vs[rt][lane];
                const Pack<W, 4> w = load<4>(B + (size_t)(nt * 16 + t16) * a.rank_pad + rt * 16 + q * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(to_f32(w.v[j]), v[j], acc, 0, 0, 0);
            }
            const int n = nt * 16 + q * 4;
            if (!mine) continue;
            if (a.vec_y && n < a.rows) {
                if (base) acc += *reinterpret_cast<const v4f *>(base + n);
                *reinterpret_cast<v4f *>(y + n) = acc;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < a.rows) y[n + j] = (base ? base[n + j] : 0.0f) + acc[j];
            }
        }
        __syncthreads();   // vs is the next adapter's
    }
}

// An adapter into its place, zeros around it, and its rank and scale.
template <typename W>
__global__ __launch_bounds__(256) void adapter_set_kernel(const W *A, int64_t lda, const W *B, int64_t ldb, int rank, float scale, int rows,
                                                          int cols, int rank_pad, int cols_pad, int rows_pad, W *to, AdapterMeta *meta)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, na = (int64_t)rank_pad * cols_pad, nb = (int64_t)rows_pad * rank_pad;
    if (i == 0) *meta = {rank, scale};
    if (i >= na + nb) return;
    W v{};
    if (i < na) {
        const int r = (int)(i / cols_pad), c = (int)(i - (int64_t)r * cols_pad);
        if (r < rank && c < cols) v = A[r * lda + c];
    } else {
        const int n = (int)((i - na) / rank_pad), r = (int)(i - na - (int64_t)n * rank_pad);
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
        static_cast<const W *>(A), lda, static_cast<const W *>(B), ldb, rank, scale, h->rows, h->cols, h->rank_pad, h->cols_pad, h->rows_pad,
        reinterpret_cast<W *>(h->data + slot * h->slot_bytes), h->meta + slot);
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
    a.rank_pad = h->rank_pad, a.cols_pad = h->cols_pad, a.rows_pad = h->rows_pad;
    a.vec_y = aligned(y, 16) && ldy % 4 == 0 && h->rows % 4 == 0 && (!base || (aligned(base, 16) && ldbase % 4 == 0));
    hipStream_t st = (hipStream_t)stream;
    if (type == EIF_HIP_F32) return launch_adapters<float>(a, h->type, st);
    return type == EIF_HIP_F16 ? launch_adapters<__half>(a, h->type, st) : launch_adapters<__hip_bfloat16>(a, h->type, st);
}

}  // extern "C"
