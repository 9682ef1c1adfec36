// Pointwise convolution / linear layer on E2M1 operands for gfx950 (msc_mx_linear):
//   out[m][n] = act(scale[n] * sum_k x[m][k]*w[n][k] + shift[n] + res[m][n])
// on v_mfma_scale_f32_16x16x128_f8f6f4: a lane feeds 32 consecutive k of one row (16 bytes of codes, one block) and that block's scale byte, so the
// stored layout is the instruction's own and nothing is re-laid out.  Products of codes are exact, the sums fp32.
//
// Operand roles.  w is the instruction's A operand (rows of the result: n), x its B operand (columns: m): a lane then holds consecutive n of one m.  The
// fragment rows are dealt out so that fragment f, row i is channel 16*(i >> 2) + 4*f + (i & 3) of a wave's 64: the four fragments of a lane make 16
// consecutive channels, whose scale / shift / res / out move in 16-byte pieces, 128 bytes of a row per wave instruction.
#include <type_traits>

#include "common.h"
#include "dma.h"
#include "msc_internal.h"
#include "mx.h"

namespace {

using namespace mx;

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct LinArgs {
    const uint8_t* x; const uint8_t* xs; const uint8_t* w; const uint8_t* ws;
    const float* scale; const float* shift; const void* res; void* out;
    long x_ld, xs_ld, w_ld, ws_ld, res_ld, out_ld, M;
    int K, N, nb, tiles_n, relu;         // nb: blocks of 32 along k
    int xs_quick, ws_quick;              // the eight scales of a step are one aligned load
};

__device__ __forceinline__ i32x8 fp4_operand(uint4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }

// CNT (a multiple of 8) consecutive channels from n: their scale / shift, and one row's results
template <typename T, int CNT, bool VEC> struct Epilogue {
    float sc[CNT], sh[CNT];
    int n, left;
    __device__ __forceinline__ Epilogue(const LinArgs& a, int n_) : n(n_), left(a.N - n_) {
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            sc[i] = a.scale && i < left ? a.scale[n + i] : 1.f;
            sh[i] = a.shift && i < left ? a.shift[n + i] : 0.f;
        }
    }
    __device__ __forceinline__ void row(const LinArgs& a, long m, const float* v) const {
        if (left <= 0) return;
#pragma unroll
        for (int h = 0; h < CNT; h += 8) {
            float r[8];
            const T* rp = (const T*)a.res + m * a.res_ld + n + h;
            if (!a.res) {
#pragma unroll
                for (int i = 0; i < 8; ++i) r[i] = 0.f;
            } else if (VEC && left >= h + 8) load8<T>(rp, r);
            else load8_some<T>(rp, left - h, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = fmaf(v[h + i], sc[h + i], sh[h + i]) + r[i];
                r[i] = a.relu && y < 0.f ? 0.f : y;            // NaN stays NaN
            }
            T* o = (T*)a.out + m * a.out_ld + n + h;
            if (VEC && left >= h + 8) store8<T>(o, r);
            else store8_some<T>(o, left - h, r);
        }
    }
};

// ------------------------------------------------------------------------------------------------ many rows
// WM x WN waves, each FM x 4 fragments: a tile of 16*WM*FM rows by 64*WN channels per block.  A step is 256 k (eight blocks, 128 bytes of codes and eight scale
// bytes) of every row, double-buffered in LDS: the codes by LDS-DMA, straight from the stored layout, the next step's requests going out before this step's
// products.  16-byte unit u of LDS row r sits at u ^ ((r >> 1) & 7) (the DMA's source is permuted, its destination is linear): the 16 rows of a fragment
// read fall into all the banks.  The scales go through registers and are dealt out as [wave row][lane group][fragment row][fragment] pairs of bytes, so
// that a lane has those of all its fragments in one read; loading them per lane from memory (two byte loads a fragment and step, 16 rows of a wave each) took
// several times as long as the products.
constexpr int UNITS = 8, ROWB = UNITS * 16;

template <typename T, int WM, int WN, int FM, bool VEC>
__global__ __launch_bounds__(WM * WN * 64, 2) void mx_gemm_kernel(LinArgs a) {
    constexpr int THREADS = WM * WN * 64, WAVES = WM * WN, FN = 4, TM = WM * FM * 16, TN = WN * 64;
    constexpr int DX = TM / 8 / WAVES, DW = TN / 8 / WAVES;            // DMA instructions (8 rows each) per wave and step
    constexpr int SCALES = (TM + TN) * ROWB, STAGE = SCALES + (TM + TN) * UNITS, NS = (TM + TN + THREADS - 1) / THREADS;
    static_assert(TM / 8 % WAVES == 0 && TN / 8 % WAVES == 0, "every wave requests");
    static_assert(2 * STAGE <= 160 * 1024, "LDS");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wid / WN, wn = wid % WN, g = lane >> 4, pl = lane & 15;
    const int tn = (int)(blockIdx.x % (unsigned)a.tiles_n);
    const long m0 = (long)(blockIdx.x / (unsigned)a.tiles_n) * TM;
    const int n0 = tn * TN;
    const int steps = (a.nb + UNITS - 1) / UNITS;
    const int last_m = (int)min((long)TM, a.M - m0) - 1, last_n = min(TN, a.N - n0) - 1;      // rows past the end: the last one again, their results are dropped

    // w's LDS row 16 f + i of a wave's 64 is channel 16*(i >> 2) + 4*f + (i & 3)
    auto channel = [](int slot) { return (slot & ~63) + 16 * ((slot & 15) >> 2) + 4 * ((slot >> 4) & 3) + (slot & 3); };
    const u32x4_t rx = make_srd(a.x + m0 * a.x_ld, (unsigned)(last_m * a.x_ld + a.nb * 16));
    const u32x4_t rw = make_srd(a.w + (long)n0 * a.w_ld, (unsigned)(last_n * a.w_ld + a.nb * 16));
    unsigned xo[DX], wo[DW];
    int xu[DX], wu[DW];
#pragma unroll
    for (int i = 0; i < DX; ++i) {
        const int r = (i * WAVES + wid) * 8 + (lane >> 3);
        xu[i] = (lane & 7) ^ ((r >> 1) & 7);
        xo[i] = (unsigned)min(r, last_m) * (unsigned)a.x_ld + xu[i] * 16;
    }
#pragma unroll
    for (int i = 0; i < DW; ++i) {
        const int r = (i * WAVES + wid) * 8 + (lane >> 3);
        wu[i] = (lane & 7) ^ ((r >> 1) & 7);
        wo[i] = (unsigned)min(channel(r), last_n) * (unsigned)a.w_ld + wu[i] * 16;
    }
    auto request = [&](int s, char* st) {                              // the codes of step s; blocks past the last one read as zeros
#pragma unroll
        for (int i = 0; i < DX; ++i) dma16(rx, st + (i * WAVES + wid) * 1024, s * UNITS + xu[i] < a.nb ? xo[i] + s * ROWB : OOB_OFF, 0);
#pragma unroll
        for (int i = 0; i < DW; ++i) dma16(rw, st + TM * ROWB + (i * WAVES + wid) * 1024, s * UNITS + wu[i] < a.nb ? wo[i] + s * ROWB : OOB_OFF, 0);
    };
    // scales: thread t moves the eight of LDS rows t, t + THREADS (x's rows, then w's)
    const uint8_t* sp[NS];
    int so[NS], sf[NS];                  // LDS place for lane group 0; bytes from lane group to lane group
    bool quick[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int r = i * THREADS + tid;
        if (r < TM) {
            sp[i] = a.xs + (m0 + min(r, last_m)) * a.xs_ld;
            so[i] = SCALES + ((r / (FM * 16) * 64 + r % 16) * FM + r % (FM * 16) / 16) * 2;
            sf[i] = FM * 32;
            quick[i] = a.xs_quick;
        } else {
            const int w = min(r - TM, TN - 1);
            sp[i] = a.ws + (long)(n0 + min(channel(w), last_n)) * a.ws_ld;
            so[i] = SCALES + TM * UNITS + ((w / 64 * 64 + w % 16) * FN + w % 64 / 16) * 2;
            sf[i] = FN * 32;
            quick[i] = a.ws_quick;
        }
    }
    uint2 rs[NS];
    auto fetch_scales = [&](int s) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i * THREADS + tid >= TM + TN) continue;
            if (quick[i]) {
                rs[i] = *reinterpret_cast<const uint2*>(sp[i] + s * UNITS);
            } else {                     // past the last block the codes are zero: any scale but the NaN one
                unsigned b[UNITS];
#pragma unroll
                for (int k = 0; k < UNITS; ++k) b[k] = s * UNITS + k < a.nb ? sp[i][s * UNITS + k] : 127u;
                rs[i] = make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
            }
        }
    };
    auto put_scales = [&](char* st) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i * THREADS + tid >= TM + TN) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) *reinterpret_cast<uint16_t*>(st + so[i] + k * sf[i]) = (uint16_t)((k < 2 ? rs[i].x : rs[i].y) >> (k & 1) * 16);
        }
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](const char* st) {
        int qx[FM / 2], qw[FN / 2];      // two fragments to a register, two bytes each
        const char* px = st + SCALES + ((wm * 4 + g) * 16 + pl) * FM * 2;
        const char* pw = st + SCALES + TM * UNITS + ((wn * 4 + g) * 16 + pl) * FN * 2;
#pragma unroll
        for (int k = 0; k < FM / 2; ++k) qx[k] = reinterpret_cast<const int*>(px)[k];
#pragma unroll
        for (int k = 0; k < FN / 2; ++k) qw[k] = reinterpret_cast<const int*>(pw)[k];
        auto half = [&](auto hh) {
            constexpr int H = decltype(hh)::value;
            uint4 fx[FM], fw[FN];
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                const int r = wn * 64 + f * 16 + pl;
                fw[f] = *reinterpret_cast<const uint4*>(st + (TM + r) * ROWB + ((2 * g + H) ^ ((r >> 1) & 7)) * 16);
            }
#pragma unroll
            for (int f = 0; f < FM; ++f) {
                const int r = wm * (FM * 16) + f * 16 + pl;
                fx[f] = *reinterpret_cast<const uint4*>(st + r * ROWB + ((2 * g + H) ^ ((r >> 1) & 7)) * 16);
            }
            // the scale's byte is an immediate: even and odd fragments apart
            auto one = [&](auto ii, auto jj, int i, int j) {
                constexpr int SX = decltype(ii)::value * 2 + H, SW = decltype(jj)::value * 2 + H;
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(fw[j]), fp4_operand(fx[i]), acc[i][j], 4, 4, SW, qw[j / 2], SX, qx[i / 2]);
            };
#pragma unroll
            for (int i = 0; i < FM; i += 2)
#pragma unroll
                for (int j = 0; j < FN; j += 2) {
                    one(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{}, i, j);
                    one(std::integral_constant<int, 0>{}, std::integral_constant<int, 1>{}, i, j + 1);
                    one(std::integral_constant<int, 1>{}, std::integral_constant<int, 0>{}, i + 1, j);
                    one(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}, i + 1, j + 1);
                }
        };
        half(std::integral_constant<int, 0>{});
        half(std::integral_constant<int, 1>{});
    };

    fetch_scales(0);
    request(0, smem);
    put_scales(smem);
    wait_vmcnt<0>();
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        char* next = smem + ((s + 1) & 1) * STAGE;                     // last read two barriers ago
        if (s + 1 < steps) {
            fetch_scales(s + 1);
            request(s + 1, next);
        }
        compute(smem + (s & 1) * STAGE);
        if (s + 1 < steps) put_scales(next);
        wait_vmcnt<0>();                 // the requests, which the compiler does not see
        __syncthreads();
    }
    // fragment f, result row 4 g + r: channel 16 g + 4 f + r of the wave's 64
    const Epilogue<T, 4 * FN, VEC> ep(a, n0 + wn * 64 + 16 * g);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = wm * (FM * 16) + i * 16 + pl;
        float v[4 * FN];
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * f + r] = acc[i][f][r];
        if (m <= last_m) ep.row(a, m0 + m, v);
    }
}

// ------------------------------------------------------------------------------------------------ few rows
// A block owns 16 channels; its eight waves share out the k range in pieces of eight blocks (a lane 32 bytes of its row of w, a wave 128 of each of 16 rows), so
// that the weights stream once through registers at full width, and add their accumulators through LDS.  FUSED (up to 16 rows): every block quantises x
// into LDS itself, in the shadow of its first weight loads -- one launch instead of two; otherwise x's codes come from memory (the caches), FM fragments of 16 rows.
constexpr int FEW_WAVES = 8, FEW_THREADS = FEW_WAVES * 64;
static int64_t few_lds(int64_t M, int64_t nb) {          // of the fused form: codes, scales and the waves' sums
    const int64_t pad = (nb + 7) / 8 * 8;
    return M * (pad * 17 + 16) + FEW_WAVES * 64 * 16;
}

template <typename T, int FM, bool FUSED> __global__ __launch_bounds__(FEW_THREADS) void mx_few_rows_kernel(LinArgs a, const T* xin, long xin_ld, int xvec) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, g = lane >> 4, pl = lane & 15;
    const int n0 = blockIdx.x * 16;
    const int nbp = (a.nb + 7) / 8 * 8, pieces = nbp / 8, pitch = nbp * 16 + 16, M = (int)a.M;
    f32x4* sums = reinterpret_cast<f32x4*>(lds);                       // [FM][waves][64]
    char* xc = lds + FEW_WAVES * 64 * 16;
    char* xsc = xc + M * pitch;                                        // (FUSED: FM = 1)
    const long row = min(n0 + pl, a.N - 1);
    const uint8_t* wr = a.w + row * a.w_ld + g * 32;
    const uint8_t* sr = a.ws + row * a.ws_ld + g * 2;

    struct Piece { uint4 w0, w1; int s; };
    auto two_scales = [&](const uint8_t* p, int b) {                   // blocks b, b + 1: zero codes past the end take any scale but the NaN one
        return (b < a.nb ? (int)p[0] : 127) | (b + 1 < a.nb ? (int)p[1] : 127) << 8;
    };
    auto load = [&](int p) {
        Piece q;
        const int b = p * 8 + 2 * g;
        q.w0 = p < pieces && b < a.nb ? *reinterpret_cast<const uint4*>(wr + (long)p * 128) : make_uint4(0, 0, 0, 0);
        q.w1 = p < pieces && b + 1 < a.nb ? *reinterpret_cast<const uint4*>(wr + (long)p * 128 + 16) : make_uint4(0, 0, 0, 0);
        q.s = p < pieces ? two_scales(sr + (long)p * 8, b) : 0x7f7f;
        return q;
    };
    Piece cur = load(wid), next = load(wid + FEW_WAVES);
    if constexpr (FUSED) {
        const int per_row = nbp * 4;
        for (int id = tid; id < M * per_row; id += FEW_THREADS) {      // whole quads
            const int m = id / per_row, k = id - m * per_row, left = a.K - k * 8;
            float v[8], q[8];
            const T* p = xin + (long)m * xin_ld + k * 8;
            if (xvec && left >= 8) load8<T>(p, v);
            else load8_some<T>(p, left, v);
            const unsigned e = block_scale<E2M1, T>(v, q);
            *reinterpret_cast<unsigned*>(xc + m * pitch + k * 4) = encode8_e2m1(q);
            if ((k & 3) == 0) xsc[m * nbp + (k >> 2)] = (char)e;
        }
        __syncthreads();
    }
    f32x4 acc[FM];
#pragma unroll
    for (int f = 0; f < FM; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int p = wid; p < pieces; p += FEW_WAVES) {
        const Piece w = cur;
        cur = next;
        next = load(p + 2 * FEW_WAVES);
        const int b = p * 8 + 2 * g;
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            uint4 x0, x1;
            int sx;
            if constexpr (FUSED) {
                const int m = min(pl, M - 1);                          // columns past the last row are dropped
                const char* xr = xc + m * pitch + b * 16;
                x0 = *reinterpret_cast<const uint4*>(xr);
                x1 = *reinterpret_cast<const uint4*>(xr + 16);
                sx = *reinterpret_cast<const uint16_t*>(xsc + m * nbp + b);
            } else {
                const long m = min(f * 16 + pl, M - 1);
                const uint8_t* xr = a.x + m * a.x_ld + (long)b * 16;
                x0 = b < a.nb ? *reinterpret_cast<const uint4*>(xr) : make_uint4(0, 0, 0, 0);
                x1 = b + 1 < a.nb ? *reinterpret_cast<const uint4*>(xr + 16) : make_uint4(0, 0, 0, 0);
                sx = two_scales(a.xs + m * a.xs_ld + b, b);
            }
            acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(w.w0), fp4_operand(x0), acc[f], 4, 4, 0, w.s, 0, sx);
            acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(w.w1), fp4_operand(x1), acc[f], 4, 4, 1, w.s, 1, sx);
        }
    }
#pragma unroll
    for (int f = 0; f < FM; ++f) sums[(f * FEW_WAVES + wid) * 64 + lane] = acc[f];
    __syncthreads();
    if (wid >= FM) return;
    f32x4 v = sums[wid * FEW_WAVES * 64 + lane];
#pragma unroll
    for (int i = 1; i < FEW_WAVES; ++i) v += sums[(wid * FEW_WAVES + i) * 64 + lane];
    const int m = wid * 16 + pl, n = n0 + 4 * g;
    if (m >= M) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (n + r >= a.N) continue;
        const float sc = a.scale ? a.scale[n + r] : 1.f, sh = a.shift ? a.shift[n + r] : 0.f;
        const float res = a.res ? ElemIO<T>::load((const T*)a.res + (long)m * a.res_ld + n + r) : 0.f;
        const float y = fmaf(v[r], sc, sh) + res;
        ElemIO<T>::store((T*)a.out + (long)m * a.out_ld + n + r, a.relu && y < 0.f ? 0.f : y);
    }
}

constexpr int FUSED_ROWS = 16, FEW_ROWS = 64;
constexpr int64_t FUSED_LDS = 64 * 1024;

struct LinPlan { int64_t nb, xc_ld, codes, scales; bool pack, fused, few; };
LinPlan lin_plan(const msc_mx_linear_desc* d) {
    LinPlan p;
    p.nb = ((int64_t)d->K + BLOCK - 1) / BLOCK;
    p.fused = d->x && d->M <= FUSED_ROWS && few_lds(d->M, p.nb) <= FUSED_LDS;
    p.few = d->M <= FEW_ROWS;
    p.pack = d->x && !p.fused;
    p.xc_ld = p.nb * E2M1::BYTES;
    p.codes = p.pack ? d->M * p.xc_ld : 0;                     // a multiple of 16
    p.scales = p.pack ? (d->M * p.nb + 15) / 16 * 16 : 0;
    return p;
}

int lin_check(const msc_mx_linear_desc* d) {
    if (!d) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: null descriptor");
    if (!msc_dtype_ok(d->dtype)) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: unknown dtype %d", d->dtype);
    if (d->M < 0 || d->K <= 0 || d->N <= 0 || d->K > (1 << 24) || d->N > (1 << 24) || d->M >= 1ll << 36)
        return msc_fail(MSC_ERR_ARG, "msc_mx_linear: bad shape (M %lld, K %d, N %d)", (long long)d->M, d->K, d->N);
    return MSC_OK;
}

template <typename T, int WM, int WN, int FM> int lin_launch(const LinArgs& a, bool vec, hipStream_t st) {
    constexpr int TM = WM * FM * 16, TN = WN * 64, LDS = 2 * (TM + TN) * (ROWB + UNITS);
    LinArgs b = a;
    b.tiles_n = (a.N + TN - 1) / TN;
    const int64_t blocks = (a.M + TM - 1) / TM * b.tiles_n;
    if (blocks >= 1ll << 31) return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_linear: 2^31 tiles or more");
    if (TM * a.x_ld >= 1ll << 31 || TN * a.w_ld >= 1ll << 31) return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_linear: a tile's rows span 2 GiB");
    auto k = vec ? mx_gemm_kernel<T, WM, WN, FM, true> : mx_gemm_kernel<T, WM, WN, FM, false>;
    if (LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return msc_fail(MSC_ERR_HIP, "msc_mx_linear: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(WM * WN * 64), LDS, st, b);
    return MSC_OK;
}
template <typename T> int lin_by_tile(const LinArgs& a, const LinPlan& p, const msc_mx_linear_desc* d, bool vec, hipStream_t st) {
    const dim3 few((unsigned)((a.N + 15) / 16));
    const long none = 0;
    if (p.fused) {
        hipLaunchKernelGGL((mx_few_rows_kernel<T, 1, true>), few, dim3(FEW_THREADS), (size_t)few_lds(a.M, a.nb), st, a, (const T*)d->x, (long)d->x_ld,
                           (int)vec_ok(d->x, d->x_ld, d->dtype));
        return MSC_OK;
    }
    if (p.few) {
        const int fm = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
        auto k = fm == 1 ? mx_few_rows_kernel<T, 1, false> : fm == 2 ? mx_few_rows_kernel<T, 2, false> : mx_few_rows_kernel<T, 4, false>;
        hipLaunchKernelGGL(k, few, dim3(FEW_THREADS), (size_t)fm * FEW_WAVES * 64 * 16, st, a, (const T*)nullptr, none, 0);
        return MSC_OK;
    }
    auto tiles = [&](int tm, int tn) { return (a.M + tm - 1) / tm * ((a.N + tn - 1) / tn); };
    if (tiles(256, 256) >= 256) return lin_launch<T, 2, 4, 8>(a, vec, st);
    if (tiles(128, 128) >= 256) return lin_launch<T, 2, 2, 4>(a, vec, st);
    return lin_launch<T, 2, 1, 2>(a, vec, st);
}

}  // namespace

extern "C" int64_t msc_mx_linear_workspace_bytes(const msc_mx_linear_desc* d) {
    if (lin_check(d)) return -1;
    const LinPlan p = lin_plan(d);
    return p.codes + p.scales;
}

extern "C" int msc_mx_linear(const msc_mx_linear_desc* d, void* stream) {
    int rc = lin_check(d);
    if (rc || d->M == 0) return rc;
    const LinPlan p = lin_plan(d);
    const int es = msc_dtype_size(d->dtype);
    if (!d->out || d->out_ld < d->N || (uintptr_t)d->out % es || (d->res && (d->res_ld < d->N || (uintptr_t)d->res % es)))
        return msc_fail(MSC_ERR_ARG, "msc_mx_linear: null or misaligned out / res, or a row pitch below %d channels", d->N);
    if (d->res == d->out && d->res_ld != d->out_ld) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: res in place needs out's row pitch");
    if (!packed_ok(d->w, d->w_ld, d->w_scales, d->s_ld, d->K, E2M1::BYTES))
        return msc_fail(MSC_ERR_ARG, "msc_mx_linear: w needs 16-byte aligned rows of whole E2M1 blocks and one scale byte per block");
    if (d->x && (d->x_ld < d->K || (uintptr_t)d->x % es))
        return msc_fail(MSC_ERR_ARG, "msc_mx_linear: x misaligned or row pitch %lld below %d channels", (long long)d->x_ld, d->K);
    LinArgs a;
    a.x = a.xs = nullptr;
    a.x_ld = a.xs_ld = 0;
    if (p.pack) {
        if (!d->ws || (uintptr_t)d->ws & 15) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: workspace missing or not 16-byte aligned");
        uint8_t* codes = (uint8_t*)d->ws;
        a.x = codes; a.x_ld = p.xc_ld; a.xs = codes + p.codes; a.xs_ld = p.nb;
        rc = msc_mx_pack(d->x, d->x_ld, d->dtype, codes, p.xc_ld, codes + p.codes, p.nb, MSC_MX_E2M1, d->M, d->K, stream);
        if (rc) return rc;
    } else if (!d->x) {
        if (!packed_ok(d->x_codes, d->xc_ld, d->x_scales, d->xs_ld, d->K, E2M1::BYTES))
            return msc_fail(MSC_ERR_ARG, "msc_mx_linear: x (or its codes: 16-byte aligned rows of whole E2M1 blocks, and scales) missing");
        a.x = d->x_codes; a.x_ld = d->xc_ld; a.xs = d->x_scales; a.xs_ld = d->xs_ld;
    }
    a.w = d->w; a.w_ld = d->w_ld; a.ws = d->w_scales; a.ws_ld = d->s_ld;
    a.scale = d->scale; a.shift = d->shift; a.res = d->res; a.out = d->out;
    a.res_ld = d->res_ld; a.out_ld = d->out_ld; a.M = d->M; a.K = d->K; a.N = d->N; a.nb = (int)p.nb; a.relu = d->relu; a.tiles_n = 0;
    auto quick = [&](const uint8_t* s, long ld) { return ((uintptr_t)s & 7) == 0 && ld % 8 == 0 && p.nb % UNITS == 0; };
    a.xs_quick = quick(a.xs, a.xs_ld); a.ws_quick = quick(a.ws, a.ws_ld);
    const bool vec = vec_ok(d->out, d->out_ld, d->dtype) && (!d->res || vec_ok(d->res, d->res_ld, d->dtype));
    hipStream_t st = (hipStream_t)stream;
    rc = d->dtype == MSC_F32 ? lin_by_tile<float>(a, p, d, vec, st) : d->dtype == MSC_BF16 ? lin_by_tile<bf16_t>(a, p, d, vec, st) : lin_by_tile<f16_t>(a, p, d, vec, st);
    return rc ? rc : msc_check_launch("msc_mx_linear");
}
