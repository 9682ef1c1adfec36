// Weight gradient of a convolution (a linear layer: 1x1) from the E4M3 checkpoint of its input, for gfx950 (msc_mx_wgrad).
//
//   dw[a][kh][kw][b] = sum_m p[m][a] * q[pixel(m)*stride - pad + (kh,kw)][b],   m over the pixels of the output grid
//
// A GEMM whose reduction runs over pixels, the outer dimension of both operands.  Per tap, a block takes a TA x TB tile of the gradient and a range of
// pixels; its steps stage KP pixels of both operands pixel-major in LDS.  The codes are turned into the compute type on the way (an E4M3 value times
// a power of two is a bf16 / fp16 / f32 number, so the matrix instructions see exactly what was stored): half the bytes of the
// 16-bit input come from HBM, and the conversion is one instruction for two elements, once per block.  The k-contiguous fragments come out of LDS by
// transposing reads.  The pixel ranges' partial tiles go to the workspace, tile by tile and coalesced, and a second launch adds them in order.
//
// What bounds it.  131072 pixels, 256 x 64: HBM (75 MB, 16.6 + 4 us with the join in the profiler, 19.6 us undisturbed = 3.9 TB/s).  32x16x16, 256 -> 256, 3x3 (9.7 GFLOP, 6 us of
// matrix instructions): latency -- nine steps a group; of 24 us some 9 are launch, first loads and partial sums, and loads, LDS writes, reads and products
// of a step take about as long as each other and overlap in part.  Divisions in the loop, the depth of the prefetch and the share of VALU
// work were tried out of it one by one: within 3 %.
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
    const float s = scale_value(e);                                    // (a pixel that was not read: codes and byte 0)
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

template <typename T, int TA, int TB, int KG, bool VECP> __global__ __launch_bounds__(KG * THREADS, 2) void mx_wgrad_kernel(WgArgs a) {
    using L = Tile<T, TA, TB>;
    constexpr int UPRA = L::PITCH_A / 16, UPRB = L::PITCH_B / 16;
    static_assert(KG == 1 || 2 * L::STAGE >= L::NF * THREADS * 16, "a group's sums fit its stages");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int grp = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, lane = tid & 63, wid = tid >> 6;
    char* const smem = lds + grp * 2 * L::STAGE;
    const int wa = wid >> 1, wb = wid & 1, g = lane >> 4, pl = lane & 15;
    // order: the tiles of one tap and one pixel range, then the taps, then the ranges.  Block b runs on XCD b % 8.  Where a few blocks read the same pixels each XCD
    // gets a run of the order, so that they share an L2 (131072 pixels, 256 x 64, two tiles: 16.5 us against 17.8); where many do, they are spread over the
    // XCDs: the same lines wanted by 36 blocks of one XCD at a time make a queue (32x16x16, 256 -> 256, 3x3: 4 us more)
    const unsigned xcd = blockIdx.x & 7, per = gridDim.x >> 3, more = gridDim.x & 7;
    const unsigned id = a.tiles * a.taps <= 8 ? xcd * per + min(xcd, more) + (blockIdx.x >> 3) : blockIdx.x;
    const unsigned bt = div_of(id, a.tile_div);
    const int tile = (int)(id - bt * a.tile_div.d);
    const int split = (int)(bt / (unsigned)a.taps), tap = (int)(bt - (unsigned)split * a.taps);
    const int a0 = tile / a.tiles_b * TA, b0 = tile % a.tiles_b * TB;
    const int kh = tap / a.KW, kw = tap - kh * a.KW;
    const int beg = split * a.chunk, mend = min(a.M, beg + a.chunk), mbeg = beg + grp * L::KP;      // the groups take turns: step i of group j is pixels KP * (KG i + j) on
    const int steps = (mend - beg + KG * L::KP - 1) / (KG * L::KP);

    struct Regs { uint4 p[L::IA], q[L::IB]; unsigned e[L::IB]; };      // what a thread moves in one step
    Regs even, odd;
    // Addresses.  The descriptors' bases move with the step (scalar), the lanes' offsets into them stay: p's rows are equally far apart, and rows past the range or
    // channels past the end read as zeros by the descriptor's extent.  q's pixel of a row, under this block's tap, advances by constants with one wrap
    // per axis; pixels outside the image read as zeros by an offset out of range.  (Divisions and 64-bit products per load and step took more issue slots
    // than the matrix instructions.)
    unsigned po[L::IA];
#pragma unroll
    for (int i = 0; i < L::IA; ++i) {
        const int idx = i * THREADS + tid, c = idx % L::UA * L::PE;
        po[i] = a0 + c < a.A ? (unsigned)(idx / L::UA) * (unsigned)(a.p_ld * L::ES) + c * L::ES : OOB_OFF;
    }
    const char* const pbase = a.p + ((long)mbeg * a.p_ld + a0) * L::ES;
    const unsigned first_n = div_of((unsigned)beg, a.hw);
    const long first_pix = a.direct ? beg : (long)first_n * a.Hq * a.Wq;
    const int pixels = a.direct ? mend - beg : (int)(div_of((unsigned)(mend - 1), a.hw) - first_n + 1) * a.Hq * a.Wq;
    const __amdgpu_buffer_rsrc_t rq_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.q + first_pix * a.q_ld), 0, (int)((pixels - 1) * a.q_ld + a.q_bytes), 0x00020000);
    const __amdgpu_buffer_rsrc_t rs_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.qs + first_pix * a.s_ld), 0, (int)((pixels - 1) * a.s_ld + a.q_bytes / BLOCK), 0x00020000);
    int qrow[L::IB], qx[L::IB], qy[L::IB], qpix[L::IB], qb[L::IB];
#pragma unroll
    for (int i = 0; i < L::IB; ++i) {
        const int idx = i * THREADS + tid, row = idx / L::UB;
        const unsigned m = (unsigned)(mbeg + row), n = div_of(m, a.hw), rem = m - n * a.hw.d, y = div_of(rem, a.w);
        qb[i] = b0 + idx % L::UB * 16;
        qrow[i] = qb[i] < a.q_bytes && !(L::B_SOME && idx >= L::KP * L::UB) ? row : 0x7fffffff;
        qy[i] = (int)y;
        qx[i] = (int)(rem - y * a.w.d);
        qpix[i] = a.direct ? grp * L::KP + row : ((int)(n - first_n) * a.Hq + qy[i] * a.stride - a.pad + kh) * a.Wq + qx[i] * a.stride - a.pad + kw;
    }
    const int Hp = (int)(a.hw.d / a.w.d), Wp = (int)a.w.d;
    const int dn = (int)div_of(KG * L::KP, a.hw), dr = KG * L::KP - dn * (int)a.hw.d, dy = (int)div_of((unsigned)dr, a.w), dx = dr - dy * Wp;
    const int dpix = a.direct ? KG * L::KP : (dn * a.Hq + dy * a.stride) * a.Wq + dx * a.stride;
    const int wrap_x = a.direct ? 0 : (a.Wq - Wp) * a.stride, wrap_y = a.direct ? 0 : (a.Hq - Hp * a.stride) * a.Wq;
    // output rows / columns whose pixel under this tap is inside the image: [lo, lo + n)
    auto first_in = [&](int k) { return (max(a.pad - k, 0) + a.stride - 1) / a.stride; };
    auto end_in = [&](int k, int in, int out) { return min(out, (in - 1 + a.pad - k) / a.stride + 1); };
    const int ylo = a.direct ? 0 : first_in(kh), yn = a.direct ? Hp : (a.Hq - 1 + a.pad - kh < 0 ? 0 : max(0, end_in(kh, a.Hq, Hp) - ylo));
    const int xlo = a.direct ? 0 : first_in(kw), xn = a.direct ? Wp : (a.Wq - 1 + a.pad - kw < 0 ? 0 : max(0, end_in(kw, a.Wq, Wp) - xlo));
    auto fetch = [&](int s, Regs& r) {                                 // in the order of the steps
        const int left = mend - mbeg - s * KG * L::KP;                 // rows; the last group's may be none
        const char* const at = pbase + (long)s * (KG * L::KP) * a.p_ld * L::ES;
        if constexpr (VECP) {
            const __amdgpu_buffer_rsrc_t rp_ = __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, left > 0 ? (int)(((min(left, L::KP) - 1) * a.p_ld + a.A - a0) * L::ES) : 0, 0x00020000);
#pragma unroll
            for (int i = 0; i < L::IA; ++i) r.p[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rp_, (int)po[i], 0, 0));
        } else {
#pragma unroll
            for (int i = 0; i < L::IA; ++i) {
                const int idx = i * THREADS + tid, row = idx / L::UA, c = a0 + idx % L::UA * L::PE;
                const char* src = at + (long)row * a.p_ld * L::ES + idx % L::UA * 16;
                r.p[i] = load_unit<T>(reinterpret_cast<const T*>(src), row < left ? a.A - c : 0);
            }
        }
#pragma unroll
        for (int i = 0; i < L::IB; ++i) {
            const bool in = qrow[i] < left && (unsigned)(qy[i] - ylo) < (unsigned)yn && (unsigned)(qx[i] - xlo) < (unsigned)xn;
            r.q[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rq_, in ? qpix[i] * (int)a.q_ld + qb[i] : (int)OOB_OFF, 0, 0));
            r.e[i] = __builtin_amdgcn_raw_buffer_load_b8(rs_, in ? qpix[i] * (int)a.s_ld + (qb[i] >> 5) : (int)OOB_OFF, 0, 0);
            qpix[i] += dpix;
            qx[i] += dx;
            const bool wx = qx[i] >= Wp;
            qx[i] -= wx ? Wp : 0;
            qy[i] += dy + (wx ? 1 : 0);
            const bool wy = qy[i] >= Hp;
            qy[i] -= wy ? Hp : 0;
            qpix[i] += (wx ? wrap_x : 0) + (wy ? wrap_y : 0);
        }
    };
    auto put = [&](char* st, const Regs& v) {
#pragma unroll
        for (int i = 0; i < L::IA; ++i) {
            const int idx = i * THREADS + tid, r = idx / L::UA, u = idx % L::UA;
            *reinterpret_cast<uint4*>(st + r * L::PITCH_A + (L::ES == 2 ? swz16<UPRA>(u, r) : u) * 16) = v.p[i];
        }
        char* sq = st + L::KP * L::PITCH_A;
#pragma unroll
        for (int i = 0; i < L::IB; ++i) {
            const int idx = i * THREADS + tid, r = idx / L::UB, u = idx % L::UB;
            if (!L::B_SOME || idx < L::KP * L::UB) stage_q<T, UPRB>(sq + r * L::PITCH_B, u, r, v.q[i], v.e[i]);
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

    // two steps' loads are in flight in registers while a third is multiplied
    fetch(0, even);
    if (steps > 1) fetch(1, odd);
    put(smem, even);
    if (steps > 2) fetch(2, even);
    __syncthreads();
    auto step = [&](int s, Regs& r) {                                  // r: step s + 1, which goes to the half that was multiplied before the last barrier
        if (s + 1 < steps) put(smem + ((s + 1) & 1) * L::STAGE, r);    // before the products, so that they cover it (3x3: 25.4 -> 23.9 us)
        if (s + 3 < steps) fetch(s + 3, r);
        compute(smem + (s & 1) * L::STAGE);
        __syncthreads();
    };
    for (int s = 0; s < steps; s += 2) {
        step(s, odd);
        if (s + 1 < steps) step(s + 1, even);
    }

    if constexpr (KG > 1) {              // the groups' sums, in order, through the stages that were multiplied last
        float4* mine = reinterpret_cast<float4*>(smem) + tid;
        if (grp) {
#pragma unroll
            for (int f = 0; f < L::NF; ++f) {
                const f32x4 v = acc[f / L::FN][f % L::FN];
                mine[f * THREADS] = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int k = 1; k < KG; ++k)
#pragma unroll
            for (int f = 0; f < L::NF; ++f) {
                const float4 v = reinterpret_cast<const float4*>(lds + k * 2 * L::STAGE)[f * THREADS + tid];
                acc[f / L::FN][f % L::FN] += f32x4{v.x, v.y, v.z, v.w};
            }
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

// adds the ranges' partial tiles, SLICES of them side by side (a fixed order); a float4 per thread, at the places the tile kernel's threads wrote
template <int TA, int TB, int SLICES> __global__ __launch_bounds__(THREADS) void mx_wgrad_join_kernel(WgArgs a) {
    constexpr int FN = TB / 32, NF = TA / 32 * FN, PLACES = THREADS / SLICES;
    __shared__ float4 red[SLICES > 1 ? THREADS : 1];
    const int slice = threadIdx.x / PLACES;
    const long at = (long)blockIdx.x * PLACES + threadIdx.x % PLACES;                  // [tap][tile][fragment][thread of the tile kernel]
    const long plane = (long)a.taps * a.tiles * NF * THREADS;
    const float4* src = reinterpret_cast<const float4*>(a.part) + at;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    int k = slice;
    for (; k + 7 * SLICES < a.splits; k += 8 * SLICES) {
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = src[(k + i * SLICES) * plane];
#pragma unroll
        for (int i = 0; i < 8; ++i) { s.x += v[i].x; s.y += v[i].y; s.z += v[i].z; s.w += v[i].w; }
    }
    for (; k < a.splits; k += SLICES) {
        const float4 v = src[k * plane];
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    if constexpr (SLICES > 1) {
        red[threadIdx.x] = s;
        __syncthreads();
        if (slice) return;
#pragma unroll
        for (int i = 1; i < SLICES; ++i) {
            const float4 v = red[i * PLACES + threadIdx.x];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
    }
    const int thread = (int)(at % THREADS), f = (int)(at / THREADS % NF), bt = (int)(at / (THREADS * NF)), tap = bt / a.tiles, tile = bt % a.tiles;
    const int lane = thread & 63, wid = thread >> 6;
    const int ia = tile / a.tiles_b * TA + (wid >> 1) * (TA / 2) + f / FN * 16 + (lane & 15);
    const int ib = tile % a.tiles_b * TB + (wid & 1) * (TB / 2) + f % FN * 16 + 4 * (lane >> 4);
    if (ia >= a.A) return;
    float* o = a.dw + ((long)ia * a.taps + tap) * a.B + ib;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (ib + i < a.B) o[i] = (a.accumulate ? o[i] : 0.f) + v[i];
}

struct WgPlan { int ta, tb, kg, tiles_a, tiles_b, splits, chunk; };
WgPlan wg_plan(const msc_mx_wgrad_desc* d) {
    WgPlan p;
    const int64_t M = (int64_t)d->N * d->Hp * d->Wp, taps = d->KH * d->KW;
    const int kp = d->dtype == MSC_F32 ? 32 : 64;
    // Tiles of 128 read less, but are few and take longer to start.  They are for 2^31 products and more where their blocks can fill the card: without splitting the pixels, or with
    // ranges that stay long.  us with the join, 128 : 64, bf16: 8192 pixels, 256 x 256, 3x3 29.8 : 50.3; 6144 27.8 : 39.3; 2048 22.5 : 17.9; 131072, 256 x 64 20.5 : 21.0;
    // 65536, 256 x 64 17.2 : 15.8; 32768, 256 x 256 21.3 : 22.9; 400, 384 x 384, 3x3 19.3 : 12.5; 4096, 128 x 512 13.6 : 11.1; 2048 pixels: 512 x 2048 22.6 : 18.4, 1024 x 2048
    // 30.3 : 25.7, 2048 x 2048 (256 blocks) 42.6 : 47.9, 512 x 512, 3x3 (144 blocks) 39.6 : 36.7.  In a graph of twelve calls, 1x1, at 2048 / 4096 / 8192 pixels: 64 blocks (1024 x 1024) 21.3 :
    // 17.1 / 28.4 : 27.7 / 41.6 : 49.0; 96 (1024 x 1536) 26.3 : 23.0 / 38.6 : 37.7 / 63.3 : 67.0; 121 30.0 : 23.5 / 43.9 : 39.4 / 70.0 : 70.4; 144 40.3 : 35.2 / 66.1 : 58.0 / 117 : 105;
    // 160 40.6 : 35.1 / 66.1 : 58.6 / 117 : 107; 192 40.6 : 35.5 / 65.7 : 59.5 / 116 : 109; 256 40.5 : 44.1 / 65.5 : 74.9 / 116 : 135.  What the rule gives away: up to 15 % at 160 to
    // some 230 blocks, which fill the card's 256 CUs in part, and up to 10 % near 4096 pixels
    const int64_t large = (int64_t)((d->A + 127) / 128) * ((d->B + 127) / 128) * taps;
    const bool wide = M * taps * d->A >= ((1ll << 31) + d->B - 1) / d->B && (large >= 160 || (large <= 128 && M >= 4096));
    p.ta = wide && d->A > 64 ? 128 : 64;
    p.tb = wide && d->B > 64 ? 128 : 64;
    p.tiles_a = (d->A + p.ta - 1) / p.ta;
    p.tiles_b = (d->B + p.tb - 1) / p.tb;
    const int64_t all = (int64_t)p.tiles_a * p.tiles_b * taps;
    // two groups of waves to a block and one block to a CU where every group has four steps to do: half the partial sums of two blocks with one group each
    // (3x3 above: 24.1 + 5.4 us to join, against 24.8 + 7.2; 1x1: 16.7 + 4.0 against 17.3 + 4.5).  Tiles of 128 always have: 2^31 products are four
    // steps for 512 groups.  Less work: more, smaller blocks
    p.kg = M * all >= 256ll * 2 * 4 * kp ? 2 : 1;
    int64_t splits = 512 / p.kg / all, most = (M + 4 * p.kg * kp - 1) / (4 * p.kg * kp);
    if (splits > most) splits = most;
    // a block's offsets into q are 32-bit: its images, one more at each end, stay below 1 GiB (a single image does, wg_check)
    const int64_t image = (int64_t)d->Hq * d->Wq * (d->q_ld > d->s_ld ? d->q_ld : d->s_ld), hw = (int64_t)d->Hp * d->Wp;
    const int64_t images = (1ll << 30) / (image > 1 ? image : 1), pixels = (images > 3 ? images - 2 : 1) * hw;
    if (splits < (M + pixels - 1) / pixels) splits = (M + pixels - 1) / pixels;
    if (splits < 1) splits = 1;
    p.chunk = (int)(((M + splits - 1) / splits + p.kg * kp - 1) / (p.kg * kp) * (p.kg * kp));
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
    const int64_t hw = (int64_t)d->Hp * d->Wp, image = (int64_t)d->Hq * d->Wq, most = 1ll << 28;      // (factors first: no product below passes 64 bits)
    if (hw >= 1ll << 30 || d->N * hw >= 1ll << 30 || image >= 1ll << 30) return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_wgrad: 2^30 pixels or more");
    if (d->q_ld >= most || d->s_ld >= most || image * d->q_ld >= most || image * d->s_ld >= most || d->p_ld >= 1ll << 24)
        return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_wgrad: an image of 2^28 bytes of codes or more, or rows of 2^24 elements");
    return MSC_OK;
}

template <typename T, int TA, int TB, int KG> int wg_launch_tiles(const WgArgs& a, bool vec, hipStream_t st) {
    constexpr int LDS = KG * 2 * Tile<T, TA, TB>::STAGE;
    auto k = vec ? mx_wgrad_kernel<T, TA, TB, KG, true> : mx_wgrad_kernel<T, TA, TB, KG, false>;
    if (LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return msc_fail(MSC_ERR_HIP, "msc_mx_wgrad: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(k, dim3((unsigned)(a.tiles * a.taps * a.splits)), dim3(KG * THREADS), LDS, st, a);
    return MSC_OK;
}
template <typename T, int TA, int TB> int wg_launch(const WgPlan& p, const WgArgs& a, bool vec, hipStream_t st) {
    int rc;
    if constexpr (TA == 64 && TB == 64) rc = p.kg == 2 ? wg_launch_tiles<T, 64, 64, 2>(a, vec, st) : wg_launch_tiles<T, 64, 64, 1>(a, vec, st);
    else rc = wg_launch_tiles<T, TA, TB, 2>(a, vec, st);
    if (rc || a.splits == 1) return rc;
    const int64_t places = (int64_t)a.tiles * a.taps * TA * TB / 4;
    // enough threads to have the partial sums' reads in flight (256 ranges of 256 x 64: 12.7 us with one slice, 4.5 with sixteen)
    if (places * 4 > 256 * THREADS || a.splits < 8) hipLaunchKernelGGL((mx_wgrad_join_kernel<TA, TB, 1>), dim3((unsigned)(places / THREADS)), dim3(THREADS), 0, st, a);
    else if (places * 16 > 256 * THREADS || a.splits < 32) hipLaunchKernelGGL((mx_wgrad_join_kernel<TA, TB, 4>), dim3((unsigned)(places / THREADS * 4)), dim3(THREADS), 0, st, a);
    else hipLaunchKernelGGL((mx_wgrad_join_kernel<TA, TB, 16>), dim3((unsigned)(places / THREADS * 16)), dim3(THREADS), 0, st, a);
    return MSC_OK;
}
template <typename T> int wg_by_tile(const WgPlan& p, const WgArgs& a, bool vec, hipStream_t st) {
    if (p.ta == 128 && p.tb == 128) return wg_launch<T, 128, 128>(p, a, vec, st);
    if (p.ta == 128) return wg_launch<T, 128, 64>(p, a, vec, st);
    if (p.tb == 128) return wg_launch<T, 64, 128>(p, a, vec, st);
    return wg_launch<T, 64, 64>(p, a, vec, st);
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
    const int64_t all = (int64_t)p.tiles_a * p.tiles_b * d->KH * d->KW;        // a launch has fewer than 2^32 threads: of the products, of the join
    if (all * p.splits >= 1ll << 23 || (p.splits > 1 && all * (p.ta / 32) * (p.tb / 32) >= 1ll << 24))
        return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_wgrad: 2^23 tiles or more");
    const int64_t hw = (int64_t)d->Hp * d->Wp, image = (int64_t)d->Hq * d->Wq * (d->q_ld > d->s_ld ? d->q_ld : d->s_ld);
    if (((p.chunk - 1) / hw + 2) * image >= 1ll << 31)
        return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_wgrad: the images of %d output pixels span 2 GiB", p.chunk);
    const int64_t dw_bytes = (int64_t)d->A * d->KH * d->KW * d->B * 4, nb = ((int64_t)d->B + BLOCK - 1) / BLOCK, q_rows = (int64_t)d->N * d->Hq * d->Wq;
    const Rows dw = one_row(d->dw, dw_bytes);
    if (meet(dw, {d->p, d->p_ld * es, (int64_t)d->A * es, d->N * hw}) || meet(dw, {d->q, d->q_ld, nb * BLOCK, q_rows}) || meet(dw, {d->q_scales, d->s_ld, nb, q_rows}))
        return msc_fail(MSC_ERR_ARG, "msc_mx_wgrad: dw shares memory with an operand");
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
    rc = d->dtype == MSC_F32 ? wg_by_tile<float>(p, a, vec, st) : d->dtype == MSC_BF16 ? wg_by_tile<bf16_t>(p, a, vec, st) : wg_by_tile<f16_t>(p, a, vec, st);
    return rc ? rc : msc_check_launch("msc_mx_wgrad");
}
