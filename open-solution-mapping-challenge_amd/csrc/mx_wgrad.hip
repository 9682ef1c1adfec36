// Weight gradient of a convolution (a linear layer: 1x1) from the E4M3 checkpoint of its input, for gfx950 (msc_mx_wgrad).
//
//   dw[a][kh][kw][b] = sum_m p[m][a] * q[pixel(m)*stride - pad + (kh,kw)][b],   m over the pixels of the output grid
//
// A GEMM whose reduction runs over pixels, the outer dimension of both operands.  Per tap, a block takes a TA x TB tile of the gradient and a range of
// pixels; its steps stage KP pixels of both operands pixel-major in LDS.  The codes are turned into the compute type on the way (an E4M3 value times
// a power of two is a bf16 / fp16 / f32 number, so the matrix instructions see exactly what was stored): half the bytes of the
// 16-bit input come from HBM, and the conversion is one instruction for two elements, once per block.  The k-contiguous fragments come out of LDS by
// transposing reads.  The pixel ranges' partial tiles go to the workspace, tile by tile and coalesced, and a second launch adds them in order.
#include <type_traits>

#include "common.h"
#include "dma.h"
#include "msc_internal.h"
#include "mx.h"

namespace {

using namespace mx;

constexpr int THREADS = 256;

struct WgArgs {
    const char* p; const uint8_t* q; const uint8_t* qs; float* dw; float* part;
    long p_ld, q_ld, s_ld;
    FastDiv hw, w, tile_div;             // pixels of an output image / row; tiles_a * tiles_b
    int Hq, Wq, A, B, KW, taps, stride, pad, M, chunk, tiles, tiles_b, splits, q_bytes, accumulate, direct;
};

typedef short v4i16_t __attribute__((ext_vector_type(4)));

// 16-byte units of a pixel row are permuted in pairs so that the eight rows a transposing read of 32 lanes touches (r .. r+3 and r+8 .. r+11, 32 bytes each) fall
// into different banks: with rows of 256 bytes the key is (r & 3) | bit 3 of r, with rows of 128 bytes the row's parity already tells two halves apart
template <int UPR> __device__ __forceinline__ int swz16(int unit, int row) {
    const int key = UPR == 16 ? (row & 3) | (((row >> 3) & 1) << 2) : ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
    return (((unit >> 1) ^ key) << 1) | (unit & 1);
}

template <typename T, int TA, int TB> struct Tile {
    static constexpr int ES = sizeof(T);
    static constexpr int KP = ES == 2 ? 64 : 32;                       // pixels per step
    static constexpr int PE = 16 / ES;                                 // elements per 16-byte unit
    static constexpr int PITCH_A = ES == 2 ? TA * 2 : TA * 4 + 64;     // bytes per LDS row: f32 rows 64 bytes apart in the banks
    static constexpr int PITCH_B = ES == 2 ? TB * 2 : TB * 4 + 64;
    static constexpr int STAGE = KP * (PITCH_A + PITCH_B);
    static constexpr int UA = TA / PE, UB = TB / 16;                   // units of a row: 16 bytes of p; 16 codes of q
    static constexpr int IA = KP * UA / THREADS;
    static constexpr int IB = KP * UB / THREADS > 0 ? KP * UB / THREADS : 1;
    static constexpr bool B_SOME = KP * UB < THREADS;
    static constexpr int FM = TA / 32, FN = TB / 32;                   // 16-wide fragments of a wave's half
    static constexpr int NF = FM * FN;
    static_assert(KP * UA % THREADS == 0 && (B_SOME || KP * UB % THREADS == 0), "units per thread");
};

// 16 codes of pixel row r, unit u of 16 -> 16 elements in LDS
template <typename T, int UPR> __device__ __forceinline__ void stage_q(char* row, int u, int r, uint4 w, unsigned e) {
    if (e == NAN_E) {                                                  // the block's 32 values are NaN: the NaN code does it
        w = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
        e = 127;
    }
    const float s = pow2_field(e);
    const unsigned c[4] = {w.x, w.y, w.z, w.w};
    if constexpr (sizeof(T) == 2) {
        unsigned o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (__is_same(T, bf16_t)) {
                o[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c[i], s, false));
                o[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c[i], s, true));
            } else {
                o[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[i], s, false));
                o[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)c[i], s, true));
            }
        }
        char* at = row + swz16<UPR>(2 * u, r) * 16;                    // a pair of units stays together
        *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(at + 16) = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[4];
            decode4_e4m3(c[i], s, v);
            *reinterpret_cast<float4*>(row + u * 64 + i * 16) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

template <typename T, int TA, int TB, bool VECP> __global__ __launch_bounds__(THREADS, 2) void mx_wgrad_kernel(WgArgs a) {
    using L = Tile<T, TA, TB>;
    constexpr int UPRA = L::PITCH_A / 16, UPRB = L::PITCH_B / 16;
    __shared__ __attribute__((aligned(16))) char smem[2 * L::STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int wa = wid >> 1, wb = wid & 1, g = lane >> 4, pl = lane & 15;
    // consecutive blocks: the tiles of one tap and one pixel range, then the taps, then the ranges -- what runs together reads the same pixels
    const unsigned bt = div_of(blockIdx.x, a.tile_div);
    const int tile = (int)(blockIdx.x - bt * a.tile_div.d);
    const int split = (int)(bt / (unsigned)a.taps), tap = (int)(bt - (unsigned)split * a.taps);
    const int a0 = tile / a.tiles_b * TA, b0 = tile % a.tiles_b * TB;
    const int kh = tap / a.KW, kw = tap - kh * a.KW;
    const int mbeg = split * a.chunk, mend = min(a.M, mbeg + a.chunk);
    const int steps = (mend - mbeg + L::KP - 1) / L::KP;

    uint4 rp[L::IA], rq[L::IB];
    unsigned re[L::IB];
    auto fetch = [&](int s) {
        const int m0 = mbeg + s * L::KP;
#pragma unroll
        for (int i = 0; i < L::IA; ++i) {
            const int idx = i * THREADS + tid, m = m0 + idx / L::UA, c = a0 + idx % L::UA * L::PE;
            const T* src = (const T*)a.p + (long)m * a.p_ld + c;
            rp[i] = make_uint4(0, 0, 0, 0);
            if (m < mend) {
                if (VECP) {
                    if (c < a.A) rp[i] = *reinterpret_cast<const uint4*>(src);          // A is a whole number of units
                } else {
                    unsigned t[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < L::PE; ++k)
                        if (c + k < a.A) {
                            if (L::ES == 2) t[k >> 1] |= (unsigned)reinterpret_cast<const uint16_t*>(src)[k] << (k & 1) * 16;
                            else t[k & 3] = reinterpret_cast<const unsigned*>(src)[k];
                        }
                    rp[i] = make_uint4(t[0], t[1], t[2], t[3]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < L::IB; ++i) {
            const int idx = i * THREADS + tid, m = m0 + idx / L::UB, b = b0 + idx % L::UB * 16;
            rq[i] = make_uint4(0, 0, 0, 0);
            re[i] = 127;
            if (m >= mend || b >= a.q_bytes || (L::B_SOME && idx >= L::KP * L::UB)) continue;
            long at = m;
            if (!a.direct) {
                const unsigned n = div_of((unsigned)m, a.hw), rem = (unsigned)m - n * a.hw.d, y = div_of(rem, a.w), x = rem - y * a.w.d;
                const int iy = (int)y * a.stride - a.pad + kh, ix = (int)x * a.stride - a.pad + kw;
                if ((unsigned)iy >= (unsigned)a.Hq || (unsigned)ix >= (unsigned)a.Wq) continue;
                at = ((long)n * a.Hq + iy) * a.Wq + ix;
            }
            rq[i] = *reinterpret_cast<const uint4*>(a.q + at * a.q_ld + b);
            re[i] = a.qs[at * a.s_ld + (b >> 5)];
        }
    };
    auto put = [&](char* st) {
#pragma unroll
        for (int i = 0; i < L::IA; ++i) {
            const int idx = i * THREADS + tid, r = idx / L::UA, u = idx % L::UA;
            *reinterpret_cast<uint4*>(st + r * L::PITCH_A + (L::ES == 2 ? swz16<UPRA>(u, r) : u) * 16) = rp[i];
        }
        char* sq = st + L::KP * L::PITCH_A;
#pragma unroll
        for (int i = 0; i < L::IB; ++i) {
            const int idx = i * THREADS + tid, r = idx / L::UB, u = idx % L::UB;
            if (!L::B_SOME || idx < L::KP * L::UB) stage_q<T, UPRB>(sq + r * L::PITCH_B, u, r, rq[i], re[i]);
        }
    };

    f32x4 acc[L::FM][L::FN];
#pragma unroll
    for (int i = 0; i < L::FM; ++i)
#pragma unroll
        for (int j = 0; j < L::FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // 16-bit: a lane of a 16-lane group addresses pixel row 8g + (pl >> 2) (+4 for the second half), channels 4*(pl & 3) .. +3, and receives four
    // pixels of channel pl
    typedef __attribute__((address_space(3))) v4i16_t* lds_v4_t;
    auto frag = [&](const char* base, int pitch, auto upr, int c, int k0) -> uint4 {
        uint2 h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = k0 + 8 * g + (pl >> 2) + 4 * i, cc = c + 4 * (pl & 3);
            h[i] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4_t)(base + r * pitch + swz16<decltype(upr)::value>(cc >> 3, r) * 16 + (cc & 7) * 2)));
        }
        return make_uint4(h[0].x, h[0].y, h[1].x, h[1].y);
    };
    auto compute = [&](const char* st) {
        const char* sq = st + L::KP * L::PITCH_A;
        const int ca = wa * (TA / 2), cb = wb * (TB / 2);
        if constexpr (L::ES == 2) {
#pragma unroll
            for (int k0 = 0; k0 < L::KP; k0 += 32) {
                uint4 fa[L::FM], fb[L::FN];
#pragma unroll
                for (int i = 0; i < L::FM; ++i) fa[i] = frag(st, L::PITCH_A, std::integral_constant<int, UPRA>{}, ca + i * 16, k0);
#pragma unroll
                for (int j = 0; j < L::FN; ++j) fb[j] = frag(sq, L::PITCH_B, std::integral_constant<int, UPRB>{}, cb + j * 16, k0);
#pragma unroll
                for (int i = 0; i < L::FM; ++i)
#pragma unroll
                    for (int j = 0; j < L::FN; ++j) Mma<T>::run(fb[j], fa[i], acc[i][j]);         // rows of the result: b, columns: a
            }
        } else {
            for (int k0 = 0; k0 < L::KP; k0 += 4) {
                float fa[L::FM], fb[L::FN];
#pragma unroll
                for (int i = 0; i < L::FM; ++i) fa[i] = *reinterpret_cast<const float*>(st + (k0 + g) * L::PITCH_A + (ca + i * 16 + pl) * 4);
#pragma unroll
                for (int j = 0; j < L::FN; ++j) fb[j] = *reinterpret_cast<const float*>(sq + (k0 + g) * L::PITCH_B + (cb + j * 16 + pl) * 4);
#pragma unroll
                for (int i = 0; i < L::FM; ++i)
#pragma unroll
                    for (int j = 0; j < L::FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j], fa[i], acc[i][j], 0, 0, 0);
            }
        }
    };

    fetch(0);
    put(smem);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) fetch(s + 1);
        compute(smem + (s & 1) * L::STAGE);
        if (s + 1 < steps) put(smem + ((s + 1) & 1) * L::STAGE);      // last read two barriers ago
        __syncthreads();
    }

    // a lane holds, of fragment (i, j): b = b0 + half + 16 j + 4 g + 0..3, a = a0 + half + 16 i + pl
    if (a.splits > 1) {
        float4* o = reinterpret_cast<float4*>(a.part) + ((long)(split * a.taps + tap) * a.tiles + tile) * (L::NF * THREADS) + tid;
#pragma unroll
        for (int f = 0; f < L::NF; ++f) {
            const f32x4 v = acc[f / L::FN][f % L::FN];
            o[f * THREADS] = make_float4(v[0], v[1], v[2], v[3]);
        }
        return;
    }
#pragma unroll
    for (int f = 0; f < L::NF; ++f) {
        const int ia = a0 + wa * (TA / 2) + f / L::FN * 16 + pl, ib = b0 + wb * (TB / 2) + f % L::FN * 16 + 4 * g;
        if (ia >= a.A) continue;
        float* o = a.dw + ((long)ia * a.taps + tap) * a.B + ib;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (ib + k < a.B) o[k] = (a.accumulate ? o[k] : 0.f) + acc[f / L::FN][f % L::FN][k];
    }
}

// adds the ranges' partial tiles in order; one float4 per thread, at the place the tile kernel's thread wrote it
template <int TA, int TB> __global__ __launch_bounds__(THREADS) void mx_wgrad_join_kernel(WgArgs a) {
    constexpr int FN = TB / 32, NF = TA / 32 * FN;
    const int bt = blockIdx.x / NF, f = blockIdx.x % NF, tap = bt / a.tiles, tile = bt % a.tiles;
    const long plane = (long)a.taps * a.tiles * NF * THREADS;
    const float4* src = reinterpret_cast<const float4*>(a.part) + ((long)bt * NF + f) * THREADS + threadIdx.x;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    int k = 0;
    for (; k + 8 <= a.splits; k += 8) {
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = src[(k + i) * plane];
#pragma unroll
        for (int i = 0; i < 8; ++i) { s.x += v[i].x; s.y += v[i].y; s.z += v[i].z; s.w += v[i].w; }
    }
    for (; k < a.splits; ++k) {
        const float4 v = src[k * plane];
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int ia = tile / a.tiles_b * TA + (wid >> 1) * (TA / 2) + f / FN * 16 + (lane & 15);
    const int ib = tile % a.tiles_b * TB + (wid & 1) * (TB / 2) + f % FN * 16 + 4 * (lane >> 4);
    if (ia >= a.A) return;
    float* o = a.dw + ((long)ia * a.taps + tap) * a.B + ib;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (ib + i < a.B) o[i] = (a.accumulate ? o[i] : 0.f) + v[i];
}

struct WgPlan { int ta, tb, tiles_a, tiles_b, splits, chunk; };
WgPlan wg_plan(const msc_mx_wgrad_desc* d) {
    WgPlan p;
    p.ta = d->A > 64 ? 128 : 64;
    p.tb = d->B > 64 ? 128 : 64;
    p.tiles_a = (d->A + p.ta - 1) / p.ta;
    p.tiles_b = (d->B + p.tb - 1) / p.tb;
    const int64_t M = (int64_t)d->N * d->Hp * d->Wp, all = (int64_t)p.tiles_a * p.tiles_b * d->KH * d->KW;
    const int kp = d->dtype == MSC_F32 ? 32 : 64;
    int64_t splits = 512 / all, most = (M + 4 * kp - 1) / (4 * kp);       // two blocks per CU, at least four steps each
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.chunk = (int)(((M + splits - 1) / splits + kp - 1) / kp * kp);
    p.splits = (int)((M + p.chunk - 1) / p.chunk);
    return p;
}

int wg_check(const msc_mx_wgrad_desc* d) {
    if (!d) return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: null descriptor");
    if (!msc_dtype_ok(d->dtype)) return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: unknown dtype %d", d->dtype);
    if (d->N < 0 || d->Hp <= 0 || d->Wp <= 0 || d->A <= 0 || d->Hq <= 0 || d->Wq <= 0 || d->B <= 0 || d->A > (1 << 20) || d->B > (1 << 20))
        return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: bad shape");
    if (d->KH <= 0 || d->KW <= 0 || d->KH > 16 || d->KW > 16 || d->stride <= 0 || d->stride > 16 || d->pad < 0 || d->pad > 16)
        return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: kernel %dx%d, stride %d, padding %d", d->KH, d->KW, d->stride, d->pad);
    if ((int64_t)d->N * d->Hp * d->Wp >= 1ll << 30 || (int64_t)d->Hq * d->Wq >= 1ll << 30)
        return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_wgrad: 2^30 pixels or more");
    return MSC_OK;
}

template <typename T, int TA, int TB> void wg_launch(const WgArgs& a, bool vec, hipStream_t st) {
    const dim3 grid((unsigned)(a.tiles * a.taps * a.splits));
    hipLaunchKernelGGL((vec ? mx_wgrad_kernel<T, TA, TB, true> : mx_wgrad_kernel<T, TA, TB, false>), grid, dim3(THREADS), 0, st, a);
    if (a.splits > 1)
        hipLaunchKernelGGL((mx_wgrad_join_kernel<TA, TB>), dim3((unsigned)(a.tiles * a.taps * (TA / 32) * (TB / 32))), dim3(THREADS), 0, st, a);
}
template <typename T> void wg_by_tile(const WgPlan& p, const WgArgs& a, bool vec, hipStream_t st) {
    if (p.ta == 128 && p.tb == 128) wg_launch<T, 128, 128>(a, vec, st);
    else if (p.ta == 128) wg_launch<T, 128, 64>(a, vec, st);
    else if (p.tb == 128) wg_launch<T, 64, 128>(a, vec, st);
    else wg_launch<T, 64, 64>(a, vec, st);
}

}  // namespace

extern "C" int64_t msc_mx_wgrad_workspace_bytes(const msc_mx_wgrad_desc* d) {
    if (wg_check(d)) return -1;
    if (d->N == 0) return 0;
    const WgPlan p = wg_plan(d);
    return p.splits == 1 ? 0 : (int64_t)p.splits * d->KH * d->KW * p.tiles_a * p.tiles_b * p.ta * p.tb * 4;
}

extern "C" int msc_mx_wgrad(const msc_mx_wgrad_desc* d, void* stream) {
    int rc = wg_check(d);
    if (rc) return rc;
    if (d->N == 0) {                     // a sum over nothing
        if (!d->dw) return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: null tensor");
        return d->accumulate ? MSC_OK : msc_memset_zero(d->dw, (int64_t)d->A * d->KH * d->KW * d->B * 4, stream);
    }
    const int es = msc_dtype_size(d->dtype);
    if (!d->p || !d->dw || d->p_ld < d->A || (uintptr_t)d->p % es || (uintptr_t)d->dw & 3)
        return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: null or misaligned tensor, or row pitch %lld below %d channels", (long long)d->p_ld, d->A);
    if (!packed_ok(d->q, d->q_ld, d->q_scales, d->s_ld, d->B, E4M3::BYTES))
        return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: q needs 16-byte aligned rows of whole E4M3 blocks and one scale byte per block");
    const WgPlan p = wg_plan(d);
    if (p.splits > 1 && (!d->ws || (uintptr_t)d->ws & 15)) return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: workspace missing or not 16-byte aligned");
    if ((int64_t)p.tiles_a * p.tiles_b * d->KH * d->KW * (p.ta / 32) * (p.tb / 32) >= 1ll << 30)
        return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_wgrad: gradient of more than 2^40 elements");
    WgArgs a;
    a.p = (const char*)d->p; a.q = d->q; a.qs = d->q_scales; a.dw = d->dw; a.part = (float*)d->ws;
    a.p_ld = d->p_ld; a.q_ld = d->q_ld; a.s_ld = d->s_ld;
    a.hw = fast_div((unsigned)(d->Hp * d->Wp)); a.w = fast_div((unsigned)d->Wp); a.tile_div = fast_div((unsigned)(p.tiles_a * p.tiles_b));
    a.Hq = d->Hq; a.Wq = d->Wq; a.A = d->A; a.B = d->B; a.KW = d->KW; a.taps = d->KH * d->KW; a.stride = d->stride; a.pad = d->pad;
    a.M = d->N * d->Hp * d->Wp; a.chunk = p.chunk; a.tiles = p.tiles_a * p.tiles_b; a.tiles_b = p.tiles_b; a.splits = p.splits;
    a.q_bytes = (d->B + BLOCK - 1) / BLOCK * BLOCK; a.accumulate = d->accumulate;
    a.direct = a.taps == 1 && d->stride == 1 && d->pad == 0 && d->Hq == d->Hp && d->Wq == d->Wp;
    const bool vec = vec_ok(d->p, d->p_ld, d->dtype) && d->A % msc_dtype_vec(d->dtype) == 0;
    hipStream_t st = (hipStream_t)stream;
    if (d->dtype == MSC_F32) wg_by_tile<float>(p, a, vec, st);
    else if (d->dtype == MSC_BF16) wg_by_tile<bf16_t>(p, a, vec, st);
    else wg_by_tile<f16_t>(p, a, vec, st);
    return msc_check_launch("msc_mx_wgrad");
}
