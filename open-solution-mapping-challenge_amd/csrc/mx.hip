// Microscaled storage for gfx950: packing and restoring (msc_mx_pack / msc_mx_unpack) and the BatchNorm backward from an E4M3 checkpoint
// (msc_mx_bn_bwd).  All three stream their operands once (the BatchNorm twice: its sums come before its result); HBM bounds them.
#include <stdlib.h>

#include "common.h"
#include "msc_internal.h"
#include "mx.h"

namespace {

using namespace mx;

constexpr int THREADS = 256, UNROLL = 4, SPAN = THREADS * UNROLL;
constexpr int64_t MAX_CHUNKS = 1ll << 30;      // 8-channel chunks of one launch: chunk numbers stay below 2^31; more rows are further launches

// ------------------------------------------------------------------------------------------------ pack
// A lane takes 8 consecutive channels of a row, a quad of lanes a block: the maximum over the block is two DPP steps, loads (16 bytes a lane for the
// 16-bit types) and code stores (8 or 4 bytes) are contiguous over the wave.  Four chunks per lane are in flight.  131072 x 256 bf16 to E4M3: 102 MB in 18.0 us (5.7 TB/s), back
// 15.7 us (6.5 TB/s: writes go faster); a large copy reaches 4.7-5.0, one that the last-level cache holds 8.
template <typename F, typename T>
__global__ void pack_kernel(const T* __restrict__ x, long x_ld, uint8_t* __restrict__ codes, long codes_ld, uint8_t* __restrict__ scales, long scales_ld,
                            unsigned chunks, FastDiv per_row, int C) {
    const unsigned first = blockIdx.x * (unsigned)SPAN + threadIdx.x;
    Chunk<T> in[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const unsigned id = first + u * THREADS;
        const unsigned row = div_of(id, per_row), k = id - row * per_row.d;
        in[u] = load_chunk<T>(x + (long)row * x_ld + k * 8, id < chunks ? C - (int)(k * 8) : 0);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const unsigned id = first + u * THREADS;
        const unsigned row = div_of(id, per_row), k = id - row * per_row.d;
        float v[8], q[8];
        in[u].floats(v);
        const unsigned e = block_scale<F, T>(v, q);
        if (id >= chunks) continue;              // whole quads: `chunks` is a multiple of four
        uint8_t* c = codes + (long)row * codes_ld + k * (F::BYTES / 4);
        if (F::ID == 0) *reinterpret_cast<uint2*>(c) = encode8_e4m3(q);
        else *reinterpret_cast<unsigned*>(c) = encode8_e2m1(q);
        if ((k & 3) == 0) scales[(long)row * scales_ld + (k >> 2)] = (uint8_t)e;
    }
}

template <typename F, typename T>
__global__ void unpack_kernel(const uint8_t* __restrict__ codes, long codes_ld, const uint8_t* __restrict__ scales, long scales_ld, T* __restrict__ out,
                              long out_ld, unsigned chunks, FastDiv per_row, int C) {
    const unsigned first = blockIdx.x * (unsigned)SPAN + threadIdx.x;
    uint2 w[UNROLL];
    unsigned e[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const unsigned id = min(first + u * THREADS, chunks - 1);
        const unsigned row = div_of(id, per_row), k = id - row * per_row.d;
        const uint8_t* c = codes + (long)row * codes_ld + k * (F::BYTES / 4);
        if (F::ID == 0) w[u] = *reinterpret_cast<const uint2*>(c);
        else w[u].x = *reinterpret_cast<const unsigned*>(c);
        e[u] = scales[(long)row * scales_ld + (k >> 2)];
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const unsigned id = first + u * THREADS;
        if (id >= chunks) continue;
        const unsigned row = div_of(id, per_row), k = id - row * per_row.d;
        const float s = scale_value(e[u]);
        float v[8];
        if (F::ID == 0) { decode4_e4m3(w[u].x, s, v); decode4_e4m3(w[u].y, s, v + 4); }
        else decode8_e2m1(w[u].x, s, v);
        store_chunk<T>(out + (long)row * out_ld + k * 8, C - (int)(k * 8), v);
    }
}

template <typename F, typename T>
void launch_pack(const void* x, long x_ld, uint8_t* codes, long codes_ld, uint8_t* scales, long scales_ld, unsigned chunks, unsigned per_row, int C,
                 hipStream_t st) {
    const dim3 grid((chunks + SPAN - 1) / SPAN);
    hipLaunchKernelGGL((pack_kernel<F, T>), grid, dim3(THREADS), 0, st, (const T*)x, x_ld, codes, codes_ld, scales, scales_ld, chunks, fast_div(per_row), C);
}
template <typename F, typename T>
void launch_unpack(const uint8_t* codes, long codes_ld, const uint8_t* scales, long scales_ld, void* out, long out_ld, unsigned chunks, unsigned per_row, int C,
                   hipStream_t st) {
    const dim3 grid((chunks + SPAN - 1) / SPAN);
    hipLaunchKernelGGL((unpack_kernel<F, T>), grid, dim3(THREADS), 0, st, codes, codes_ld, scales, scales_ld, (T*)out, out_ld, chunks, fast_div(per_row), C);
}

int mx_check(const char* name, const void* x, int64_t x_ld, int dtype, const void* codes, int64_t codes_ld, const void* scales, int64_t scales_ld, int fmt,
             int64_t rows, int C) {
    if (fmt != MSC_MX_E4M3 && fmt != MSC_MX_E2M1) return msc_fail(MSC_ERR_ARG, "%s: unknown format %d", name, fmt);
    if (!msc_dtype_ok(dtype)) return msc_fail(MSC_ERR_ARG, "%s: unknown dtype %d", name, dtype);
    if (rows < 0 || C <= 0 || C > (1 << 24)) return msc_fail(MSC_ERR_ARG, "%s: bad shape (%lld rows, %d channels)", name, (long long)rows, C);
    if (rows == 0) return MSC_OK;
    if (!x || x_ld < C) return msc_fail(MSC_ERR_ARG, "%s: null tensor or row pitch %lld below %d channels", name, (long long)x_ld, C);
    if ((uintptr_t)x % msc_dtype_size(dtype)) return msc_fail(MSC_ERR_ARG, "%s: tensor not aligned to its elements", name);
    if (!packed_ok(codes, codes_ld, scales, scales_ld, C, fmt == MSC_MX_E4M3 ? E4M3::BYTES : E2M1::BYTES))
        return msc_fail(MSC_ERR_ARG, "%s: codes need 16-byte aligned rows of whole blocks, scales one byte per block (row pitches %lld / %lld, %d channels)", name,
                        (long long)codes_ld, (long long)scales_ld, C);
    const int es = msc_dtype_size(dtype);
    const int64_t nb = ((int64_t)C + BLOCK - 1) / BLOCK;
    const Rows t{x, x_ld * es, (int64_t)C * es, rows};
    if (meet(t, {codes, codes_ld, nb * (fmt == MSC_MX_E4M3 ? E4M3::BYTES : E2M1::BYTES), rows}) || meet(t, {scales, scales_ld, nb, rows}))
        return msc_fail(MSC_ERR_ARG, "%s: the tensor shares memory with its codes or scales", name);
    return MSC_OK;
}

}  // namespace

#define MX_BY_TYPE(F, call)                                              \
    do {                                                                 \
        if (dtype == MSC_F32) call<F, float> MX_ARGS;                    \
        else if (dtype == MSC_BF16) call<F, bf16_t> MX_ARGS;             \
        else call<F, f16_t> MX_ARGS;                                     \
    } while (0)

extern "C" int msc_mx_pack(const void* x, int64_t x_ld, int dtype, uint8_t* codes, int64_t codes_ld, uint8_t* scales, int64_t scales_ld, int fmt, int64_t rows,
                           int C, void* stream) {
    int rc = mx_check("msc_mx_pack", x, x_ld, dtype, codes, codes_ld, scales, scales_ld, fmt, rows, C);
    if (rc || rows == 0) return rc;
    const unsigned per_row = (unsigned)((C + BLOCK - 1) / BLOCK) * 4;
    const int64_t rows_max = MAX_CHUNKS / per_row;
    for (int64_t r = 0; r < rows; r += rows_max) {
        const int64_t n = rows - r < rows_max ? rows - r : rows_max;
        const char* xr = (const char*)x + r * x_ld * msc_dtype_size(dtype);
#define MX_ARGS (xr, x_ld, codes + r * codes_ld, codes_ld, scales + r * scales_ld, scales_ld, (unsigned)(n * per_row), per_row, C, (hipStream_t)stream)
        if (fmt == MSC_MX_E4M3) MX_BY_TYPE(E4M3, launch_pack);
        else MX_BY_TYPE(E2M1, launch_pack);
#undef MX_ARGS
    }
    return msc_check_launch("msc_mx_pack");
}

extern "C" int msc_mx_unpack(const uint8_t* codes, int64_t codes_ld, const uint8_t* scales, int64_t scales_ld, int fmt, void* out, int64_t out_ld, int dtype,
                             int64_t rows, int C, void* stream) {
    int rc = mx_check("msc_mx_unpack", out, out_ld, dtype, codes, codes_ld, scales, scales_ld, fmt, rows, C);
    if (rc || rows == 0) return rc;
    const unsigned per_row = (unsigned)((C + BLOCK - 1) / BLOCK) * 4;
    const int64_t rows_max = MAX_CHUNKS / per_row;
    for (int64_t r = 0; r < rows; r += rows_max) {
        const int64_t n = rows - r < rows_max ? rows - r : rows_max;
        char* o = (char*)out + r * out_ld * msc_dtype_size(dtype);
#define MX_ARGS (codes + r * codes_ld, codes_ld, scales + r * scales_ld, scales_ld, o, out_ld, (unsigned)(n * per_row), per_row, C, (hipStream_t)stream)
        if (fmt == MSC_MX_E4M3) MX_BY_TYPE(E4M3, launch_unpack);
        else MX_BY_TYPE(E2M1, launch_unpack);
#undef MX_ARGS
    }
    return msc_check_launch("msc_mx_unpack");
}

// ------------------------------------------------------------------------------------------------ BatchNorm backward
// More than BN_FEW rows: three launches.  reduce: a block takes every n-th few rows and up to 256 channels (a lane 8 of them), sums dh and dh*(y - mean) in fp32 over its rows, in
// double over its row groups, and leaves one partial per channel.  finish: adds the blocks' partials in order (double), writes dgamma / dbeta and the
// coefficients of dy = a*dh + c2*(y - mean) + c1.  apply: streams again.  Centring y by the batch mean before the products keeps the sum from losing what
// a large mean would cancel.
namespace {

// Rows in flight per thread, and blocks.  131072 x 256 bf16 join: reduce 34.6 us with one row, 31 with two or four (3.4 TB/s: a plain read-only sum of 1 GB reaches 4.0
// on the card), 36 with half the blocks; apply 51 with one, 42 with two (the second reading of dout and y is from the last-level cache), 40 with 4096 blocks instead of 2048, 48 with
// 8192; the rows from the end, or on the XCD that summed them: no difference.
constexpr int BN_ROWS = 4, BN_APPLY_ROWS = 2, BN_BLOCKS = 1024, BN_APPLY_BLOCKS = 4096;
constexpr int BN_COLS = 32;                    // 8-channel chunks of a block's column range at most

struct BnArgs {
    const void* dout; const uint8_t* y; const uint8_t* y_scales; const uint8_t* mask;
    const float* mean; const float* invstd; const float* gamma; const float* scale; const float* shift;
    float* dgamma; float* dbeta; void* dy; void* dres;
    double2* part; float4* coef;
    long dout_ld, y_ld, s_ld, mask_ld, dy_ld, dres_ld, rows;
    int C, strips, cols_log2, accumulate, dres_acc;
};

// what one chunk (8 channels of a row) reads, and its masked gradients and centred inputs: apart, so that several rows' loads are in flight
template <typename T> struct BnRaw { Chunk<T> d; uint2 y; unsigned e, bits; };
template <typename T, int RELU> __device__ __forceinline__ void bn_read(const BnArgs& a, long row, int c0, int left, BnRaw<T>& r) {
    r.d = load_chunk<T>((const T*)a.dout + row * a.dout_ld + c0, left);
    r.y = *reinterpret_cast<const uint2*>(a.y + row * a.y_ld + c0);
    r.e = a.y_scales[row * a.s_ld + (c0 >> 5)];
    r.bits = 0xff;
    if (RELU == 3) {
        const uint8_t* m = a.mask + row * a.mask_ld;
        if (sizeof(T) == 2) r.bits = m[c0 >> 3];
        else r.bits = (m[c0 >> 2] & 15u) | (left > 4 ? (unsigned)m[(c0 >> 2) + 1] << 4 : 0u);
    }
}
template <typename T, int RELU> __device__ __forceinline__ void bn_terms(const BnRaw<T>& r, const float* mean, const float* sc, const float* sh, float* dh, float* t) {
    const float s = scale_value(r.e);
    float y[8];
    decode4_e4m3(r.y.x, s, y);
    decode4_e4m3(r.y.y, s, y + 4);
    r.d.floats(dh);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (RELU == 2) dh[i] = fmaf(sc[i], y[i], sh[i]) > 0.f ? dh[i] : 0.f;
        if (RELU == 3) dh[i] = (r.bits >> i) & 1 ? dh[i] : 0.f;
        t[i] = y[i] - mean[i];
    }
}

template <typename T, int RELU> __global__ __launch_bounds__(256) void bn_reduce_kernel(BnArgs a) {
    __shared__ float2 red[THREADS][9];         // 8 channels per thread, one column of padding
    const int cols = 1 << a.cols_log2;
    const int col = threadIdx.x & (cols - 1), rg = threadIdx.x >> a.cols_log2, groups = THREADS >> a.cols_log2;
    const int c0 = (blockIdx.y * cols + col) * 8, left = a.C - c0;
    float s1[8], s2[8], mean[8], sc[8], sh[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s1[i] = s2[i] = 0.f;
        mean[i] = i < left ? a.mean[c0 + i] : 0.f;
        sc[i] = RELU == 2 && i < left ? a.scale[c0 + i] : 0.f;
        sh[i] = RELU == 2 && i < left ? a.shift[c0 + i] : 0.f;
    }
    auto add = [&](const BnRaw<T>& raw) {
        float dh[8], t[8];
        bn_terms<T, RELU>(raw, mean, sc, sh, dh, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) { s1[i] += dh[i]; s2[i] = fmaf(dh[i], t[i], s2[i]); }
    };
    if (left > 0) {
        for (long r = (long)blockIdx.x * BN_ROWS * groups + rg; r < a.rows; r += (long)a.strips * BN_ROWS * groups) {
            if (r + (BN_ROWS - 1) * groups < a.rows) {
                BnRaw<T> raw[BN_ROWS];
#pragma unroll
                for (int k = 0; k < BN_ROWS; ++k) bn_read<T, RELU>(a, r + k * groups, c0, left, raw[k]);
#pragma unroll
                for (int k = 0; k < BN_ROWS; ++k) add(raw[k]);
            } else {
                for (int k = 0; k < BN_ROWS && r + k * groups < a.rows; ++k) {
                    BnRaw<T> raw;
                    bn_read<T, RELU>(a, r + k * groups, c0, left, raw);
                    add(raw);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) red[threadIdx.x][i] = make_float2(s1[i], s2[i]);
    __syncthreads();
    for (int c = threadIdx.x; c < cols * 8; c += THREADS) {
        const int ch = blockIdx.y * cols * 8 + c;
        double2 s = make_double2(0.0, 0.0);
        for (int g = 0; g < groups; ++g) {
            const float2 v = red[(g << a.cols_log2) + (c >> 3)][c & 7];
            s.x += v.x; s.y += v.y;
        }
        if (ch < a.C) a.part[(long)blockIdx.x * a.C + ch] = s;
    }
}

// of one channel, from its sums (dh, dh*(y - mean)): dgamma and dbeta go out, {a, c1, c2, mean} comes back
__device__ __forceinline__ float4 bn_coefficients(const BnArgs& a, int ch, double2 s) {
    const double inv = a.invstd[ch], n = (double)a.rows;
    const double db = s.x, dg = s.y * inv, ga = (a.gamma ? (double)a.gamma[ch] : 1.0) * inv;
    if (a.dgamma) a.dgamma[ch] = (a.accumulate ? a.dgamma[ch] : 0.f) + (float)dg;
    if (a.dbeta) a.dbeta[ch] = (a.accumulate ? a.dbeta[ch] : 0.f) + (float)db;
    return make_float4((float)ga, (float)(-ga * db / n), (float)(-ga * inv * dg / n), a.mean[ch]);
}

// FIN channels x THREADS / FIN slices of the strips per block
constexpr int FIN = 4;
__global__ __launch_bounds__(256) void bn_finish_kernel(BnArgs a) {
    __shared__ double2 red[THREADS];
    constexpr int SLICES = THREADS / FIN;
    const int c = threadIdx.x % FIN, k = threadIdx.x / FIN, ch = blockIdx.x * FIN + c;
    double2 s = make_double2(0.0, 0.0);
    if (ch < a.C) {
        int i = k;
        for (; i + 7 * SLICES < a.strips; i += 8 * SLICES) {
            double2 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = a.part[(long)(i + u * SLICES) * a.C + ch];
#pragma unroll
            for (int u = 0; u < 8; ++u) { s.x += v[u].x; s.y += v[u].y; }
        }
        for (; i < a.strips; i += SLICES) {
            const double2 v = a.part[(long)i * a.C + ch];
            s.x += v.x; s.y += v.y;
        }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    for (int h = SLICES / 2; h; h >>= 1) {
        if (k < h) {
            const double2 v = red[threadIdx.x + h * FIN];
            s.x += v.x; s.y += v.y;
            red[threadIdx.x] = s;
        }
        __syncthreads();
    }
    if (k || ch >= a.C) return;
    a.coef[ch] = bn_coefficients(a, ch, s);
}

// the results of one chunk
template <typename T, int RELU>
__device__ __forceinline__ void bn_store(const BnArgs& a, long r, int c0, int left, const BnRaw<T>& raw, const float4* f, const float* mean, const float* sc, const float* sh) {
    float dh[8], t[8];
    bn_terms<T, RELU>(raw, mean, sc, sh, dh, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = fmaf(f[i].x, dh[i], fmaf(f[i].z, t[i], f[i].y));
    T* o = (T*)a.dy + r * a.dy_ld + c0;
    if (a.dres) {
        T* g = (T*)a.dres + r * a.dres_ld + c0;
        if (a.dres_acc) {
            float old[8];
            load_chunk<T>(g, left).floats(old);
#pragma unroll
            for (int i = 0; i < 8; ++i) dh[i] += old[i];
        }
        store_chunk<T>(g, left, dh);
    }
    store_chunk<T>(o, left, t);
}

template <typename T, int RELU> __global__ __launch_bounds__(256) void bn_apply_kernel(BnArgs a) {
    const int cols = 1 << a.cols_log2;
    const int col = threadIdx.x & (cols - 1), rg = threadIdx.x >> a.cols_log2, groups = THREADS >> a.cols_log2;
    const int c0 = (blockIdx.y * cols + col) * 8, left = a.C - c0;
    if (left <= 0) return;
    float4 f[8];
    float mean[8], sc[8], sh[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f[i] = i < left ? a.coef[c0 + i] : make_float4(0.f, 0.f, 0.f, 0.f);
        mean[i] = f[i].w;
        sc[i] = RELU == 2 && i < left ? a.scale[c0 + i] : 0.f;
        sh[i] = RELU == 2 && i < left ? a.shift[c0 + i] : 0.f;
    }
    for (long r = (long)blockIdx.x * BN_APPLY_ROWS * groups + rg; r < a.rows; r += (long)gridDim.x * BN_APPLY_ROWS * groups) {
        if (r + (BN_APPLY_ROWS - 1) * groups < a.rows) {               // (all the rows' loads before the first store: the outputs may be dout itself)
            BnRaw<T> raw[BN_APPLY_ROWS];
#pragma unroll
            for (int k = 0; k < BN_APPLY_ROWS; ++k) bn_read<T, RELU>(a, r + k * groups, c0, left, raw[k]);
#pragma unroll
            for (int k = 0; k < BN_APPLY_ROWS; ++k) bn_store<T, RELU>(a, r + k * groups, c0, left, raw[k], f, mean, sc, sh);
        } else {
            for (int k = 0; k < BN_APPLY_ROWS && r + k * groups < a.rows; ++k) {
                BnRaw<T> raw;
                bn_read<T, RELU>(a, r + k * groups, c0, left, raw);
                bn_store<T, RELU>(a, r + k * groups, c0, left, raw, f, mean, sc, sh);
            }
        }
    }
}

// Few rows: one launch.  A block has 16 channels and every row, kept in registers between the sums and the result: nothing is read twice, nothing is joined across
// blocks.  One launch against three, us on the device (bf16, a graph of twelve calls), without a join: 1024 x 512 7.0 : 9.4, 1536 x 512 8.0 : 9.6, 2048 x 512 8.9 : 9.8,
// 2048 x 1024 9.7 : 12.6, 2048 x 2048 14.1 : 17.3; with one: 512 x 256 6.8 : 9.7, 1024 x 512 8.9 : 10.0, 1536 x 512 10.9 : 10.2, 2048 x 256 11.7 : 10.0, 2048 x 512 12.8 : 10.8, 2048 x 1024
// 15.4 : 13.6, 1536 x 2048 15.6 : 16.5, 2048 x 2048 18.9 : 18.9.  From some 1500 rows on a join is up to 2 us better off with three, and a call from the host 5 us worse off (no workspace
// to allocate here, one launch): the limit stays one number.  A CU's lines bound the kernel: 2048 rows, one line each of dout, y and the results for 32 bytes of it.
constexpr int BN_FEW_THREADS = 512, BN_FEW_COLS = 2, BN_FEW_GROUPS = BN_FEW_THREADS / BN_FEW_COLS, BN_FEW_PER = 8, BN_FEW = BN_FEW_GROUPS * BN_FEW_PER;

template <typename T, int RELU> __global__ __launch_bounds__(BN_FEW_THREADS) void bn_few_rows_kernel(BnArgs a) {
    __shared__ float2 red[BN_FEW_THREADS][9];
    __shared__ double2 part[BN_FEW_THREADS];
    __shared__ float4 coef[16];
    const int col = threadIdx.x % BN_FEW_COLS, rg = threadIdx.x / BN_FEW_COLS;
    // block b runs on XCD b % 8: neighbours in the channels share 128-byte lines and so an XCD's L2 (2048 x 512 fp16: 14.1 -> 9.6 us)
    const unsigned xcd = blockIdx.x & 7, per = gridDim.x >> 3, more = gridDim.x & 7;
    const int place = (int)(xcd * per + min(xcd, more) + (blockIdx.x >> 3));
    const int c0 = (place * BN_FEW_COLS + col) * 8, left = a.C - c0;
    float mean[8], sc[8], sh[8], s1[8], s2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s1[i] = s2[i] = 0.f;
        mean[i] = i < left ? a.mean[c0 + i] : 0.f;
        sc[i] = RELU == 2 && i < left ? a.scale[c0 + i] : 0.f;
        sh[i] = RELU == 2 && i < left ? a.shift[c0 + i] : 0.f;
    }
    BnRaw<T> raw[BN_FEW_PER];
    if (left > 0) {
#pragma unroll
        for (int k = 0; k < BN_FEW_PER; ++k) bn_read<T, RELU>(a, min((long)rg + k * BN_FEW_GROUPS, a.rows - 1), c0, left, raw[k]);       // (no branch between the loads)
    }
#pragma unroll
    for (int k = 0; k < BN_FEW_PER; ++k) {
        if (rg + k * BN_FEW_GROUPS >= a.rows || left <= 0) continue;
        float dh[8], t[8];
        bn_terms<T, RELU>(raw[k], mean, sc, sh, dh, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) { s1[i] += dh[i]; s2[i] = fmaf(dh[i], t[i], s2[i]); }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) red[threadIdx.x][i] = make_float2(s1[i], s2[i]);
    __syncthreads();
    {                                              // 16 channels x 32 slices of the row groups
        const int c = threadIdx.x % 16, slice = threadIdx.x / 16;
        double2 s = make_double2(0.0, 0.0);
#pragma unroll
        for (int k = 0; k < BN_FEW_GROUPS / 32; ++k) {
            const float2 v = red[(slice * (BN_FEW_GROUPS / 32) + k) * BN_FEW_COLS + c / 8][c % 8];
            s.x += v.x; s.y += v.y;
        }
        part[threadIdx.x] = s;
        __syncthreads();
#pragma unroll
        for (int h = 16; h; h >>= 1) {
            if (slice < h) {
                const double2 v = part[threadIdx.x + h * 16];
                s.x += v.x; s.y += v.y;
                part[threadIdx.x] = s;
            }
            __syncthreads();
        }
        const int ch = place * 16 + c;
        if (slice == 0) coef[c] = ch < a.C ? bn_coefficients(a, ch, s) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    if (left <= 0) return;
    float4 f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = coef[col * 8 + i];
#pragma unroll
    for (int k = 0; k < BN_FEW_PER; ++k)
        if (rg + k * BN_FEW_GROUPS < a.rows) bn_store<T, RELU>(a, rg + k * BN_FEW_GROUPS, c0, left, raw[k], f, mean, sc, sh);
}

constexpr int64_t BN_ROWS_END = 1ll << 40;         // past any memory; the plan's sums stay far from 64 bits
struct BnPlan { int cols_log2, ctiles, strips, apply_strips; };
BnPlan bn_plan(int64_t rows, int C) {
    BnPlan p;
    const int chunks = (C + 7) / 8;
    p.cols_log2 = 0;
    while ((1 << p.cols_log2) < chunks && (1 << p.cols_log2) < BN_COLS) ++p.cols_log2;
    p.ctiles = (chunks + (1 << p.cols_log2) - 1) >> p.cols_log2;
    const int groups = THREADS >> p.cols_log2;
    auto strips = [&](long blocks, int each) {
        const long most = (rows + groups * each - 1) / (groups * each), n = blocks / p.ctiles;
        return (int)(n > most ? most : n < 1 ? 1 : n);
    };
    p.strips = strips(BN_BLOCKS, BN_ROWS);
    p.apply_strips = strips(BN_APPLY_BLOCKS, BN_APPLY_ROWS);
    return p;
}

template <typename T, int RELU> void bn_launch(const BnArgs& a, const BnPlan& p, hipStream_t st) {
    if (a.rows <= BN_FEW) {
        hipLaunchKernelGGL((bn_few_rows_kernel<T, RELU>), dim3((a.C + 15) / 16), dim3(BN_FEW_THREADS), 0, st, a);
        return;
    }
    const dim3 grid(p.strips, p.ctiles), apply_grid(p.apply_strips, p.ctiles);
    hipLaunchKernelGGL((bn_reduce_kernel<T, RELU>), grid, dim3(THREADS), 0, st, a);
    hipLaunchKernelGGL(bn_finish_kernel, dim3((a.C + FIN - 1) / FIN), dim3(THREADS), 0, st, a);
    hipLaunchKernelGGL((bn_apply_kernel<T, RELU>), apply_grid, dim3(THREADS), 0, st, a);
}
template <typename T> void bn_by_relu(int relu, const BnArgs& a, const BnPlan& p, hipStream_t st) {
    if (relu == 0) bn_launch<T, 0>(a, p, st);
    else if (relu == 2) bn_launch<T, 2>(a, p, st);
    else bn_launch<T, 3>(a, p, st);
}

}  // namespace

extern "C" int64_t msc_mx_bn_bwd_workspace_bytes(int64_t rows, int C) {
    if (rows <= BN_FEW || rows >= BN_ROWS_END || C <= 0 || C > (1 << 24)) return 0;
    return (int64_t)C * 16 * (1 + bn_plan(rows, C).strips);
}

extern "C" int msc_mx_bn_bwd(const msc_mx_bn_bwd_desc* d, void* stream) {
    if (!d) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: null descriptor");
    if (!msc_dtype_ok(d->dtype)) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: unknown dtype %d", d->dtype);
    if (d->rows <= 0 || d->rows >= BN_ROWS_END || d->C <= 0 || d->C > (1 << 24))
        return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: bad shape (%lld rows, %d channels)", (long long)d->rows, d->C);
    if (!d->dout || !d->dy || !d->mean || !d->invstd || (!d->ws && d->rows > BN_FEW)) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: null pointer");
    if (d->relu != 0 && d->relu != 2 && d->relu != 3) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: relu is 0, 2 or 3, got %d", d->relu);
    if (d->relu == 2 && (!d->scale || !d->shift)) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: relu 2 needs scale and shift");
    const int per = msc_dtype_vec(d->dtype);
    if (d->relu == 3 && (!d->relu_mask || d->mask_ld < (d->C + per - 1) / per))
        return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: relu 3 needs the byte mask, %d bytes per row", (d->C + per - 1) / per);
    if (d->dout_ld < d->C || d->dy_ld < d->C || (d->dres && d->dres_ld < d->C)) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: row pitch below %d channels", d->C);
    if (!packed_ok(d->y, d->y_ld, d->y_scales, d->s_ld, d->C, E4M3::BYTES))
        return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: y needs 16-byte aligned rows of whole E4M3 blocks and one scale byte per block");
    if ((uintptr_t)d->ws & 15) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: workspace not 16-byte aligned");
    const int es = msc_dtype_size(d->dtype);
    if ((uintptr_t)d->dout % es || (uintptr_t)d->dy % es || (uintptr_t)d->dres % es) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: tensor not aligned to its elements");
    if ((d->dy == d->dout && d->dy_ld != d->dout_ld) || (d->dres == d->dout && d->dres_ld != d->dout_ld) || d->dres == d->dy)
        return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: dy and dres are different buffers; either may be dout, with its row pitch");
    const BnPlan p = bn_plan(d->rows, d->C);
    if (p.ctiles > 65535) return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_bn_bwd: too many channels");
    const int64_t len = (int64_t)d->C * es, nb = ((int64_t)d->C + BLOCK - 1) / BLOCK;
    const Rows dout{d->dout, d->dout_ld * es, len, d->rows}, y{d->y, d->y_ld, nb * BLOCK, d->rows}, ys{d->y_scales, d->s_ld, nb, d->rows};
    const Rows mask{d->relu == 3 ? d->relu_mask : nullptr, d->mask_ld, (d->C + per - 1) / per, d->rows};
    const Rows dy{d->dy, d->dy_ld * es, len, d->rows}, dres{d->dres, d->dres_ld * es, len, d->rows};
    for (const Rows& o : {dy, dres})
        if ((o.p != d->dout && meet(o, dout)) || meet(o, y) || meet(o, ys) || meet(o, mask))
            return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: dy or dres shares memory with an operand and is not dout itself");
    if (meet(dy, dres)) return msc_fail(MSC_ERR_ARG, "msc_mx_bn_bwd: dy and dres share memory");
    BnArgs a;
    a.dout = d->dout; a.y = d->y; a.y_scales = d->y_scales; a.mask = d->relu_mask;
    a.mean = d->mean; a.invstd = d->invstd; a.gamma = d->gamma; a.scale = d->scale; a.shift = d->shift;
    a.dgamma = d->dgamma; a.dbeta = d->dbeta; a.dy = d->dy; a.dres = d->dres;
    a.coef = (float4*)d->ws; a.part = (double2*)((char*)d->ws + (int64_t)d->C * 16);
    a.dout_ld = d->dout_ld; a.y_ld = d->y_ld; a.s_ld = d->s_ld; a.mask_ld = d->mask_ld; a.dy_ld = d->dy_ld; a.dres_ld = d->dres_ld;
    a.rows = d->rows; a.C = d->C; a.strips = p.strips; a.cols_log2 = p.cols_log2; a.accumulate = d->accumulate; a.dres_acc = d->dres_acc;
    hipStream_t st = (hipStream_t)stream;
    if (d->dtype == MSC_F32) bn_by_relu<float>(d->relu, a, p, st);
    else if (d->dtype == MSC_BF16) bn_by_relu<bf16_t>(d->relu, a, p, st);
    else bn_by_relu<f16_t>(d->relu, a, p, st);
    return msc_check_launch("msc_mx_bn_bwd");
}
