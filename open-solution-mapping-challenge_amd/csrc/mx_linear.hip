// Pointwise convolution / linear layer on E2M1 operands for gfx950 (msc_mx_linear):
//   out[m][n] = act(scale[n] * sum_k x[m][k]*w[n][k] + shift[n] + res[m][n])
// on v_mfma_scale_f32_16x16x128_f8f6f4: a lane feeds 32 consecutive k of one row (16 bytes of codes, one block) and that block's scale byte, so the
// stored layout is the instruction's own and nothing is re-laid out.  Products of codes are exact, the sums fp32.
//
// Operand roles.  w is the instruction's A operand (rows of the result: n), x its B operand (columns: m): a lane then holds consecutive n of one m, and the
// fragment rows are dealt out so that its fragments make two runs of eight channels, which move in 16-byte pieces.
//
// Three forms: up to 16 rows (64 of a long reduction, or packed), the weights streamed once by blocks of 16 channels; up to 64 rows of a short one, or a few tiles'
// channels, x quantised by the tile kernel itself; else packing,
// then tiles of 256 x 256 (fewer: 128 x 128, 64 x 64).
//
// What bounds them.  1 x 4096 -> 4096: 5.7 us on the device for 9 MB, one wave's chain of loads; the call takes 8.5 us of host time.  8192 x 1024 -> 256: 11.8 us for
// 21 MB, the chain of a step (read, quantise, LDS, products) on two blocks per CU.  8192 x 4096 -> 4096 with a residual: 124 us, 17 of them packing (275 GFLOP:
// 2.2 PFLOP/s).  Taken apart, the product's requests alone take 49 us (512 tiles of 1.1 MB = 0.57 GB from the L2s, 11.6 TB/s), reads and products 45, the epilogue some
// 40: 134 MB of residual and result, moved by all CUs in step, with no registers left to hold a tile back (256 in use) -- together 134 for a kernel of 113 to 119,
// so that the three hardly overlap.  Requesting the residual ahead of the last step spilled (160-180 us); waiting before the stores instead of behind them, 136.
//
// Next to the 16-bit 1x1 convolution (msc_conv_igemm at its best configuration, bf16, a graph of twelve calls, us): ahead where weights or products dominate, 1 x 4096 -> 4096 5.7
// : 15.6, 8192 x 4096 -> 4096 with a residual 124 : 246; behind on a ResNet's own layers, whose x and out travel in 16 bits either way: 131072 x 64 -> 256 36.6 : 24.4,
// 131072 x 256 -> 64 27.0 : 17.4, 32768 x 512 -> 128 15.2 : 10.5, 8192 x 1024 -> 256 11.6 : 9.2, 2048 x 512 -> 2048 with a residual 13.6 : 11.2.  There it saves memory, not time.
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
    int K, N, nb, tiles_m, tiles_n, relu;         // nb: blocks of 32 along k
};

__device__ __forceinline__ i32x8 fp4_operand(uint4 v) { return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }

// eight consecutive channels from n: their scale / shift; one row's residual, and its results.  Apart, because res may be out: a loop that loads and stores row by
// row could not have the next row's load in flight
template <typename T> struct Epilogue {
    float sc[8], sh[8];
    int n, left;
    __device__ __forceinline__ Epilogue(const LinArgs& a, int n_) : n(n_), left(a.N - n_) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sc[i] = a.scale && i < left ? a.scale[n + i] : 1.f;
            sh[i] = a.shift && i < left ? a.shift[n + i] : 0.f;
        }
    }
    __device__ __forceinline__ Chunk<T> load(const LinArgs& a, long m, bool in) const { return load_chunk<T>((const T*)a.res + m * a.res_ld + n, a.res && in ? left : 0); }
    __device__ __forceinline__ void store(const LinArgs& a, long m, bool in, const Chunk<T>& res, const float* v) const {
        if (left <= 0 || !in) return;
        float r[8];
        res.floats(r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = fmaf(v[i], sc[i], sh[i]) + r[i];
            r[i] = a.relu && y < 0.f ? 0.f : y;                        // NaN stays NaN
        }
        store_chunk<T>((T*)a.out + m * a.out_ld + n, left, r);
    }
};

// ------------------------------------------------------------------------------------------------ many rows
// WM x WN waves, each FM x 4 fragments: a tile of 16*WM*FM rows by 64*WN channels at a time, a block takes several.  A step is 256 k (eight blocks: 128 bytes
// of codes and eight of scales) of every row, filled into one half of LDS by LDS-DMA straight from the stored layout while the other is multiplied; the first step
// of the next tile goes out before the last one of this tile, so that it lands during the products and the epilogue.  16-byte unit u of LDS row r sits at
// u ^ ((r >> 1) & 7) (the DMA's source is permuted, its destination is linear) and lane group g takes the units g and g + 4: the 16 lanes that a 16-byte read
// serves together (rows 0-3 and 12-15 of one group, 4-11 of the next) then fall into 16 different bank quads.  (Units 2g and 2g + 1 made them collide in
// pairs: SQ_LDS_BANK_CONFLICT was 48 % of SQ_LDS_IDX_ACTIVE.)  Scales by the dword, too: byte loads per lane and fragment took several times the products'
// time, a detour through registers a tenth of it.
constexpr int UNITS = 8, ROWB = UNITS * 16;

// 4 bytes per lane from buffer offset `voff` to LDS bytes [lds_wave_base, +256)
__device__ __forceinline__ void dma4(u32x4_t srd, char* lds_wave_base, unsigned voff) {
    const unsigned lds_addr = (unsigned)(size_t)(lds_ptr_t)lds_wave_base;
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 2\n\tbuffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds_addr), "v"(voff), "s"(srd)
                 : "memory");
}

// w's LDS row 16 f + i of a wave's 64 is this channel of its 64: a lane's fragments 0, 1 and 2, 3 are eight consecutive channels each, 64 bytes of a 16-bit row
// over the four lane groups
__device__ __forceinline__ int lin_channel(int slot) { return (slot & ~63) + 32 * (slot >> 5 & 1) + 8 * ((slot & 15) >> 2) + 4 * (slot >> 4 & 1) + (slot & 3); }

// one step's products of a wave: FM fragments of rows from LDS row wm * FM * 16, four of channels from LDS row TM + wn * 64
template <int FM, int TM> __device__ __forceinline__ void lin_step(const LinArgs& a, int s, const char* st, int SCALES, int wm, int wn, int g, int pl, f32x4 (&acc)[FM][4]) {
    constexpr int FN = 4;
    int qx[2][FM], qw[2][FN];        // byte 0: the scale of unit g / g + 4
    const char* pws = st + SCALES + (TM + wn * 64 + pl) * 8;
    const char* pxs = st + SCALES + (wm * (FM * 16) + pl) * 8;
    auto both = [&](const char* p, int& q0, int& q1) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        q0 = (int)(v.x >> 8 * g);
        q1 = (int)(v.y >> 8 * g);
    };
#pragma unroll
    for (int f = 0; f < FN; ++f) both(pws + f * 128, qw[0][f], qw[1][f]);
#pragma unroll
    for (int f = 0; f < FM; ++f) both(pxs + f * 128, qx[0][f], qx[1][f]);
    if (s * UNITS + UNITS > a.nb) {  // past the last block the codes are zero: any scale but the NaN one
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool past = s * UNITS + 4 * h + g >= a.nb;
#pragma unroll
            for (int f = 0; f < FN; ++f) qw[h][f] = past ? 127 : qw[h][f];
#pragma unroll
            for (int f = 0; f < FM; ++f) qx[h][f] = past ? 127 : qx[h][f];
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint4 fx[FM], fw[FN];
#pragma unroll
        for (int f = 0; f < FN; ++f) {
            const int r = wn * 64 + f * 16 + pl;
            fw[f] = *reinterpret_cast<const uint4*>(st + (TM + r) * ROWB + ((g + 4 * h) ^ ((r >> 1) & 7)) * 16);
        }
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            const int r = wm * (FM * 16) + f * 16 + pl;
            fx[f] = *reinterpret_cast<const uint4*>(st + r * ROWB + ((g + 4 * h) ^ ((r >> 1) & 7)) * 16);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(fw[j]), fp4_operand(fx[i]), acc[i][j], 4, 4, 0, qw[h][j], 0, qx[h][i]);
    }
}

// ... and their results.  Fragments 2h, 2h + 1 of a lane are channels 32 h + 8 g .. + 7 of the wave's 64, of row pl: stored as they are, an instruction would write 64
// bytes of each of 16 rows.  Neighbours pl, pl ^ 1 swap halves first: the even lane takes channels 8 g of both rows, the odd lane channels 32 + 8 g, and an
// instruction writes whole 128-byte lines of eight rows (131072 x 64 -> 256: 28.0 ->
// 25.8 us)
template <typename T, int FM>
__device__ __forceinline__ void lin_write(const LinArgs& a, long m0, int last_m, int n0, int wm, int wn, int g, int pl, const f32x4 (&acc)[FM][4]) {
    const bool odd = pl & 1;
    const Epilogue<T> ep(a, n0 + wn * 64 + (odd ? 32 : 0) + 8 * g);
    constexpr int ROWS = FM < 4 ? FM : 4;
#pragma unroll
    for (int i0 = 0; i0 < FM; i0 += ROWS) {
        Chunk<T> r0[ROWS], r1[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int m = wm * (FM * 16) + (i0 + k) * 16 + (pl & ~1);
            r0[k] = ep.load(a, m0 + m, m <= last_m);
            r1[k] = ep.load(a, m0 + m + 1, m + 1 <= last_m);
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int i = i0 + k, m = wm * (FM * 16) + i * 16 + (pl & ~1);
            float v0[8], v1[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float lo = acc[i][c / 4][c % 4], hi = acc[i][2 + c / 4][c % 4];
                const float got = __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(odd ? lo : hi), 0xB1, 0xF, 0xF, true));      // quad_perm [1,0,3,2]
                v0[c] = odd ? got : lo;
                v1[c] = odd ? hi : got;
            }
            ep.store(a, m0 + m, m <= last_m, r0[k], v0);
            ep.store(a, m0 + m + 1, m + 1 <= last_m, r1[k], v1);
        }
    }
}

template <typename T, int WM, int WN, int FM>
__global__ __launch_bounds__(WM * WN * 64, 2) void mx_gemm_kernel(LinArgs a) {
    constexpr int WAVES = WM * WN, FN = 4, TM = WM * FM * 16, TN = WN * 64, ROWS = TM + TN;
    constexpr int DX = TM / 8 / WAVES, DW = TN / 8 / WAVES;            // DMA instructions (8 rows of codes each) per wave and step
    constexpr int DSX = (TM / 32 + WAVES - 1) / WAVES, DSW = (TN / 32 + WAVES - 1) / WAVES;      // ... of scales (32 rows); a wave past the last repeats it
    constexpr int SCALES = ROWS * ROWB, STAGE = SCALES + ROWS * 8;
    static_assert(TM / 8 % WAVES == 0 && TN / 8 % WAVES == 0 && TM % 32 == 0, "every wave requests");
    static_assert(2 * STAGE <= 160 * 1024, "LDS");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wid / WN, wn = wid % WN, g = lane >> 4, pl = lane & 15;
    const int steps = (a.nb + UNITS - 1) / UNITS;
    // (The order of the tiles over the XCDs and the place in k where each starts were tried both ways: within 2 % of each other.)
    const unsigned tiles = (unsigned)a.tiles_m * (unsigned)a.tiles_n;

    struct Place { long m0; int n0, last_m, last_n; };
    auto place = [&](unsigned id) {
        Place p;
        p.m0 = (long)(id / (unsigned)a.tiles_n) * TM;
        p.n0 = (int)(id % (unsigned)a.tiles_n) * TN;
        p.last_m = (int)min((long)TM, a.M - p.m0) - 1;                 // rows past the end: the last one again, their results are dropped
        p.last_n = min(TN, a.N - p.n0) - 1;
        return p;
    };
    u32x4_t rx, rw, rxs, rws;
    unsigned xo[DX], wo[DW], xso[DSX], wso[DSW];
    const int u = (lane & 7) ^ ((wid * 8 + (lane >> 3)) >> 1 & 7);     // of the lane's rows, 8 * WAVES apart: one key where WAVES is even
    static_assert(WAVES % 2 == 0, "unit key");
    auto aim = [&](const Place& p) {
        rx = make_srd(a.x + p.m0 * a.x_ld, (unsigned)(p.last_m * a.x_ld + a.nb * 16));
        rw = make_srd(a.w + (long)p.n0 * a.w_ld, (unsigned)(p.last_n * a.w_ld + a.nb * 16));
        rxs = make_srd(a.xs + p.m0 * a.xs_ld, (unsigned)(p.last_m * a.xs_ld + (a.nb + 3) / 4 * 4));
        rws = make_srd(a.ws + (long)p.n0 * a.ws_ld, (unsigned)(p.last_n * a.ws_ld + (a.nb + 3) / 4 * 4));
#pragma unroll
        for (int i = 0; i < DX; ++i) xo[i] = (unsigned)min((i * WAVES + wid) * 8 + (lane >> 3), p.last_m) * (unsigned)a.x_ld + u * 16;
#pragma unroll
        for (int i = 0; i < DW; ++i) wo[i] = (unsigned)min(lin_channel((i * WAVES + wid) * 8 + (lane >> 3)), p.last_n) * (unsigned)a.w_ld + u * 16;
#pragma unroll
        for (int i = 0; i < DSX; ++i) xso[i] = (unsigned)min(min(i * WAVES + wid, TM / 32 - 1) * 32 + (lane >> 1), p.last_m) * (unsigned)a.xs_ld + (lane & 1) * 4;
#pragma unroll
        for (int i = 0; i < DSW; ++i) wso[i] = (unsigned)min(lin_channel(min(i * WAVES + wid, TN / 32 - 1) * 32 + (lane >> 1)), p.last_n) * (unsigned)a.ws_ld + (lane & 1) * 4;
    };
    auto request = [&](int s, char* st) {                              // blocks past the last one read as zeros
        const bool live = s * UNITS + u < a.nb, live_s = s * UNITS + (lane & 1) * 4 < a.nb;
#pragma unroll
        for (int i = 0; i < DX; ++i) dma16(rx, st + (i * WAVES + wid) * 1024, live ? xo[i] + s * ROWB : OOB_OFF, 0);
#pragma unroll
        for (int i = 0; i < DW; ++i) dma16(rw, st + TM * ROWB + (i * WAVES + wid) * 1024, live ? wo[i] + s * ROWB : OOB_OFF, 0);
#pragma unroll
        for (int i = 0; i < DSX; ++i) dma4(rxs, st + SCALES + min(i * WAVES + wid, TM / 32 - 1) * 256, live_s ? xso[i] + s * UNITS : OOB_OFF);
#pragma unroll
        for (int i = 0; i < DSW; ++i) dma4(rws, st + SCALES + TM * 8 + min(i * WAVES + wid, TN / 32 - 1) * 256, live_s ? wso[i] + s * UNITS : OOB_OFF);
    };

    f32x4 acc[FM][FN];
    Place here = place(blockIdx.x);
    aim(here);
    int half = 0;
    request(0, smem);
    for (unsigned id = blockIdx.x; id < tiles; id += gridDim.x) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const Place next = place(min(id + gridDim.x, tiles - 1));
        for (int s = 0; s < steps; ++s) {
            wait_vmcnt<0>();                                           // this wave's requests of this step have landed ...
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // ... its reads of the last one are done ...
            raw_barrier();                                             // ... and so for the others: the other half is free
            if (s + 1 < steps) {
                request(s + 1, smem + (half ^ 1) * STAGE);
            } else if (id + gridDim.x < tiles) {
                aim(next);
                request(0, smem + (half ^ 1) * STAGE);
            }
            lin_step<FM, TM>(a, s, smem + half * STAGE, SCALES, wm, wn, g, pl, acc);
            half ^= 1;
        }
        lin_write<T, FM>(a, here.m0, here.last_m, here.n0, wm, wn, g, pl, acc);
        here = next;
    }
}

// ------------------------------------------------------------------------------------------------ few channels
// The same tile, with x quantised on the way into LDS instead of by a launch of its own: for weights of a few tiles' channels, where every row of x is then
// quantised once or a few times.  x comes through registers (a quad of lanes a block, as in packing), w by LDS-DMA.  WM x WN = 4 waves, FM fragments of rows each.
template <typename T, int WM, int WN, int FM>
__global__ __launch_bounds__(256, 2) void mx_fused_kernel(LinArgs a, const T* xin, long xin_ld) {
    constexpr int WAVES = 4, FN = 4, TM = WM * FM * 16, TN = WN * 64, ROWS = TM + TN, DW = TN / 8 / WAVES;
    constexpr int SCALES = ROWS * ROWB, STAGE = SCALES + ROWS * 8, CHUNKS = TM * UNITS * 4 / 256;
    static_assert(WM * WN == WAVES && TN <= 256 && 2 * STAGE <= 80 * 1024, "a row of scales per thread, two blocks per CU");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wid / WN, wn = wid % WN, g = lane >> 4, pl = lane & 15;
    const int steps = (a.nb + UNITS - 1) / UNITS;
    const long m0 = (long)(blockIdx.x / (unsigned)a.tiles_n) * TM;
    const int n0 = (int)(blockIdx.x % (unsigned)a.tiles_n) * TN;
    const int last_m = (int)min((long)TM, a.M - m0) - 1, last_n = min(TN, a.N - n0) - 1;
    const u32x4_t rw = make_srd(a.w + (long)n0 * a.w_ld, (unsigned)(last_n * a.w_ld + a.nb * 16));
    const int u = (lane & 7) ^ ((wid * 8 + (lane >> 3)) >> 1 & 7);
    unsigned wo[DW];
#pragma unroll
    for (int i = 0; i < DW; ++i) wo[i] = (unsigned)min(lin_channel((i * WAVES + wid) * 8 + (lane >> 3)), last_n) * (unsigned)a.w_ld + u * 16;
    auto request = [&](int s, char* st) {
        const bool live = s * UNITS + u < a.nb;
#pragma unroll
        for (int i = 0; i < DW; ++i) dma16(rw, st + TM * ROWB + (i * WAVES + wid) * 1024, live ? wo[i] + s * ROWB : OOB_OFF, 0);
    };
    // chunk i of thread t: eight channels, number t % 32 of a step, of row t / 32 + 8 i
    const int xr = tid >> 5, xc = tid & 31;
    Chunk<T> xv[CHUNKS];
    // w's scales come through registers too, a row per thread: eight bytes at any alignment (odd row pitches need no launch that lays them out)
    typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(1), may_alias));
    const uint8_t* const wsr = a.ws + (long)(n0 + min(lin_channel(tid), last_n)) * a.ws_ld;
    uint2 sv = make_uint2(0, 0);
    auto fetch = [&](int s) {
        const int k = s * (UNITS * BLOCK) + xc * 8;
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) xv[i] = load_chunk<T>(xin + (m0 + min(xr + 8 * i, last_m)) * xin_ld + k, a.K - k);
        const int blocks = a.nb - s * UNITS;
        const uint8_t* const p = wsr + s * UNITS;
        if (blocks >= UNITS) {
            sv = __builtin_bit_cast(uint2, *reinterpret_cast<const u32x2_any*>(p));
        } else {
            unsigned e[UNITS];
#pragma unroll
            for (int i = 0; i < UNITS; ++i) e[i] = p[min(i, blocks - 1)];
            sv = make_uint2(e[0] | e[1] << 8 | e[2] << 16 | e[3] << 24, e[4] | e[5] << 8 | e[6] << 16 | e[7] << 24);
        }
    };
    auto put = [&](char* st) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const int r = xr + 8 * i, b = xc >> 2;
            float v[8], q[8];
            xv[i].floats(v);
            const unsigned e = block_scale<E2M1, T>(v, q);
            *reinterpret_cast<unsigned*>(st + r * ROWB + (b ^ ((r >> 1) & 7)) * 16 + (xc & 3) * 4) = encode8_e2m1(q);
            if ((xc & 3) == 0) st[SCALES + r * 8 + b] = (char)e;
        }
        if (tid < TN) *reinterpret_cast<uint2*>(st + SCALES + (TM + tid) * 8) = sv;
    };
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    fetch(0);
    request(0, smem);
    put(smem);
    for (int s = 0; s < steps; ++s) {
        char* const now = smem + (s & 1) * STAGE;
        char* const next = smem + ((s + 1) & 1) * STAGE;
        wait_vmcnt<0>();                                               // the requests of step s, which the compiler does not see
        __syncthreads();                                               // ... and everyone's, x's codes among them; the other half is free
        if (s + 1 < steps) {
            fetch(s + 1);
            request(s + 1, next);
        }
        lin_step<FM, TM>(a, s, now, SCALES, wm, wn, g, pl, acc);
        if (s + 1 < steps) put(next);
    }
    lin_write<T, FM>(a, m0, last_m, n0, wm, wn, g, pl, acc);
}

// scales in rows a multiple of four bytes apart, for the kernel above
__global__ __launch_bounds__(256) void mx_scale_rows_kernel(const uint8_t* __restrict__ in, long in_ld, uint8_t* __restrict__ out, long out_ld, long rows, int nb) {
    for (long row = blockIdx.x * 4l + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4l)
        for (int b = threadIdx.x & 63; b < nb; b += 64) out[row * out_ld + b] = in[row * in_ld + b];
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

template <typename T, int FM, bool FUSED> __global__ __launch_bounds__(FEW_THREADS) void mx_few_rows_kernel(LinArgs a, const T* xin, long xin_ld) {
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
            const int m = id / per_row, k = id - m * per_row;
            float v[8], q[8];
            load_chunk<T>(xin + (long)m * xin_ld + k * 8, a.K - k * 8).floats(v);
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
// x quantised by the tile kernel itself (mx_fused_kernel): for up to 64 rows of a short reduction, for weights of at most two waves' channels, and where 512 blocks of 16 (32) x 256 cover the result and the
// reduction is short.  Measured against packing first, us on the device: 8192 x 1024 -> 256 12.4 : 17.5; 131072 x 256 -> 64 27.5 : 42.0; 32768 x 512 -> 128 15.7 : 21.9;
// 2048 x 512 -> 2048 12.7 : 15.3; but 8192 x 1024 -> 1024 31.7 : 26.9, 1024 x 4096 -> 1024 29.5 : 22.4, 8192 x 4096 -> 512 48.4 : 43.2, 131072 x 64 -> 256 58.8 : 38.3
// and 24 x 1024 -> 4096 8.9 : 8.2, 64 x 1024 -> 1024 8.9 : 10.2, 64 x 256 -> 256 5.2 : 8.6, 64 x 4096 -> 128 40 : 16 (packing, then the kernel for few rows).
// Around the limit of 1024 channels, in a graph of twelve calls: 8192 x K -> 256 11.8 : 15.7 (K = 1024), 15.1 : 18.7 (1536), 18.4 : 21.5 (2048), 33.4 : 33.8 (4096); 2048 x K -> 1024
// 14.9 : 15.5 (1536), 17.9 : 16.8 (2048); 300 x K -> 512 10.7 : 11.6 (1536), 13.0 : 13.0 (2048); 512 x 2048 -> 2048 16.8 : 13.4; 40 x 1024 -> 256 8.4 : 8.7, 64 x 1536 -> 256
// 10.6 : 9.7, 24 x 2048 -> 1024 12.9 : 8.7.  The crossing lies between 1000 and 4000 with the number of channels and rows; 1024 is the side on which nothing loses
constexpr int FUSED_CHANNELS = 128, FUSED_BLOCKS = 512, FUSED_K = 1024;
constexpr int64_t FUSED_MOST = 1ll << 29;      // rows: 2^23 blocks, whose 2^31 threads are within a launch; the form behind the packing has a grid of the card's size

struct LinPlan { int64_t nb, xc_ld, s_ld, codes, scales, w_scales, bytes; bool pack, fused, few, tile; int tile_rows; };      // fused: few rows, tile: few channels -- x is quantised by the product's own launch
bool dword_rows(const void* s, int64_t ld) { return ((uintptr_t)s & 3) == 0 && ld % 4 == 0; }
LinPlan lin_plan(const msc_mx_linear_desc* d) {
    LinPlan p;
    p.nb = ((int64_t)d->K + BLOCK - 1) / BLOCK;
    p.fused = d->x && d->M <= FUSED_ROWS && few_lds(d->M, p.nb) <= FUSED_LDS;
    const int64_t tiles = (d->M + 15) / 16 * ((d->N + 255) / 256);
    p.tile_rows = tiles <= FUSED_BLOCKS ? 1 : 2;                // fragments of 16
    p.tile = d->x && !p.fused && (d->M <= FEW_ROWS ? d->K <= FUSED_K : d->M <= FUSED_MOST && (d->N <= FUSED_CHANNELS || (tiles <= 2 * FUSED_BLOCKS && d->K <= FUSED_K)));
    p.few = d->M <= FEW_ROWS && !p.tile;
    p.pack = d->x && !p.fused && !p.tile;
    p.xc_ld = p.nb * E2M1::BYTES;
    p.s_ld = (p.nb + 3) / 4 * 4;                               // rows of scales start on dwords
    p.codes = p.pack ? d->M * p.xc_ld : 0;                     // a multiple of 16
    p.scales = p.pack || !(p.few || p.tile || dword_rows(d->x_scales, d->xs_ld)) ? (d->M * p.s_ld + 15) / 16 * 16 : 0;
    p.w_scales = p.few || p.tile || dword_rows(d->w_scales, d->s_ld) ? 0 : (d->N * p.s_ld + 15) / 16 * 16;
    p.bytes = p.codes + p.scales + p.w_scales;
    return p;
}

int lin_check(const msc_mx_linear_desc* d) {
    if (!d) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: null descriptor");
    if (!msc_dtype_ok(d->dtype)) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: unknown dtype %d", d->dtype);
    if (d->M < 0 || d->K <= 0 || d->N <= 0 || d->K > (1 << 24) || d->N > (1 << 24) || d->M >= 1ll << 36)
        return msc_fail(MSC_ERR_ARG, "msc_mx_linear: bad shape (M %lld, K %d, N %d)", (long long)d->M, d->K, d->N);
    return MSC_OK;
}

// rows and channels of a block's tile (the kernels' TM, TN); 0: the form for few rows, which has none
struct LinTile { int m, n; };
LinTile lin_tile(const LinPlan& p, int64_t M, int64_t N) {
    if (p.few) return {0, 0};
    if (p.tile) {
        if (N <= 64) return {64, 64};
        if (N <= 128) return {64, 128};
        return {p.tile_rows * 16, 256};
    }
    auto tiles = [&](int t) { return (M + t - 1) / t * ((N + t - 1) / t); };
    // A larger tile reads less from the caches; a smaller one is taken while all of its tiles are resident at once (two of 128 x 128, four of 64 x 64 to a CU).  us on the
    // device, large : small: 2048 x 2048 -> 4096 (512 tiles) 30.8 : 23.0, 20480 x 2048 -> 300 (480) 31.2 : 23.6, 2304 x 2048 -> 4096 (576) 31.8 : 33.4, 3328 x 2048 -> 4096 (832) 32.6 : 38.9;
    // 2048 x 2048 -> 2048 (1024) 17.5 : 15.2, 12288 x 2048 -> 300 (960) 21.8 : 17.2, 2048 x 2048 -> 2560 (1280) 21.2 : 21.8, 1536 x 2048 -> 4096 (1536) 21.7 : 25.3
    const int t = tiles(128) > 2 * 256 ? 256 : tiles(64) > 4 * 256 ? 128 : 64;
    return {t, t};
}
// what a tile's descriptors and the grid can hold
int lin_tile_check(const LinTile& t, const LinPlan& p, const LinArgs& a) {
    if (!t.m) return MSC_OK;
    auto spans = [](int rows, int64_t ld) { return ld >= (1ll << 31) / rows; };
    if (!p.tile && (a.M + t.m - 1) / t.m * ((a.N + t.n - 1) / t.n) >= 1ll << 30) return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_linear: 2^30 tiles or more");
    if (spans(t.n, a.w_ld) || (!p.tile && (spans(t.m, a.x_ld) || spans(t.m, a.xs_ld) || spans(t.n, a.ws_ld))))
        return msc_fail(MSC_ERR_UNSUPPORTED, "msc_mx_linear: a tile's rows span 2 GiB");
    return MSC_OK;
}

template <typename T, int WM, int WN, int FM> int lin_launch(const LinArgs& a, hipStream_t st) {
    constexpr int TM = WM * FM * 16, TN = WN * 64, LDS = 2 * (TM + TN) * (ROWB + UNITS), RESIDENT = 256 * (LDS > 80 * 1024 ? 1 : LDS > 40 * 1024 ? 2 : 4);
    LinArgs b = a;
    b.tiles_n = (a.N + TN - 1) / TN;
    const int64_t tiles_m = (a.M + TM - 1) / TM, tiles = tiles_m * b.tiles_n;
    b.tiles_m = (int)tiles_m;
    auto k = mx_gemm_kernel<T, WM, WN, FM>;
    if (LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return msc_fail(MSC_ERR_HIP, "msc_mx_linear: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(k, dim3((unsigned)(tiles < RESIDENT ? tiles : RESIDENT)), dim3(WM * WN * 64), LDS, st, b);
    return MSC_OK;
}
template <typename T, int WM, int WN, int FM> int lin_launch_fused(const LinArgs& a, const msc_mx_linear_desc* d, hipStream_t st) {
    constexpr int TM = WM * FM * 16, TN = WN * 64, LDS = 2 * (TM + TN) * (ROWB + UNITS);
    LinArgs b = a;
    b.tiles_n = (a.N + TN - 1) / TN;
    const int64_t tiles = (a.M + TM - 1) / TM * b.tiles_n;
    auto k = mx_fused_kernel<T, WM, WN, FM>;
    if (LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return msc_fail(MSC_ERR_HIP, "msc_mx_linear: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(256), LDS, st, b, (const T*)d->x, (long)d->x_ld);
    return MSC_OK;
}
template <typename T> int lin_by_tile(const LinArgs& a, const LinPlan& p, const LinTile& t, const msc_mx_linear_desc* d, hipStream_t st) {
    const dim3 few((unsigned)((a.N + 15) / 16));
    const long none = 0;
    if (p.fused) {
        hipLaunchKernelGGL((mx_few_rows_kernel<T, 1, true>), few, dim3(FEW_THREADS), (size_t)few_lds(a.M, a.nb), st, a, (const T*)d->x, (long)d->x_ld);
        return MSC_OK;
    }
    if (p.few) {
        const int fm = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
        auto k = fm == 1 ? mx_few_rows_kernel<T, 1, false> : fm == 2 ? mx_few_rows_kernel<T, 2, false> : mx_few_rows_kernel<T, 4, false>;
        hipLaunchKernelGGL(k, few, dim3(FEW_THREADS), (size_t)fm * FEW_WAVES * 64 * 16, st, a, (const T*)nullptr, none);
        return MSC_OK;
    }
    if (p.tile) {
        if (t.n == 64) return lin_launch_fused<T, 4, 1, 1>(a, d, st);
        if (t.n == 128) return lin_launch_fused<T, 2, 2, 2>(a, d, st);
        if (t.m == 16) return lin_launch_fused<T, 1, 4, 1>(a, d, st);
        return lin_launch_fused<T, 1, 4, 2>(a, d, st);
    }
    if (t.m == 256) return lin_launch<T, 2, 4, 8>(a, st);
    if (t.m == 128) return lin_launch<T, 2, 2, 4>(a, st);
    return lin_launch<T, 2, 1, 2>(a, st);
}

}  // namespace

extern "C" int64_t msc_mx_linear_workspace_bytes(const msc_mx_linear_desc* d) {
    if (lin_check(d)) return -1;
    const LinPlan p = lin_plan(d);
    return p.bytes;
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
    if (d->x == d->out || d->x_codes == d->out) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: out cannot be x: other channels' blocks still read it");
    if (!d->x && !packed_ok(d->x_codes, d->xc_ld, d->x_scales, d->xs_ld, d->K, E2M1::BYTES))
        return msc_fail(MSC_ERR_ARG, "msc_mx_linear: x (or its codes: 16-byte aligned rows of whole E2M1 blocks, and scales) missing");
    if (p.bytes && (!d->ws || (uintptr_t)d->ws & 15)) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: workspace missing or not 16-byte aligned");
    LinArgs a;
    uint8_t* codes = (uint8_t*)d->ws;
    uint8_t* scales = codes + p.codes;
    uint8_t* w_scales = scales + p.scales;
    a.x = d->x_codes; a.x_ld = d->xc_ld; a.xs = d->x_scales; a.xs_ld = d->xs_ld;
    a.w = d->w; a.w_ld = d->w_ld; a.ws = d->w_scales; a.ws_ld = d->s_ld;
    if (p.pack) { a.x = codes; a.x_ld = p.xc_ld; }
    if (p.scales) { a.xs = scales; a.xs_ld = p.s_ld; }
    if (p.w_scales) { a.ws = w_scales; a.ws_ld = p.s_ld; }
    a.scale = d->scale; a.shift = d->shift; a.res = d->res; a.out = d->out;
    a.res_ld = d->res_ld; a.out_ld = d->out_ld; a.M = d->M; a.K = d->K; a.N = d->N; a.nb = (int)p.nb; a.relu = d->relu; a.tiles_m = a.tiles_n = 0;
    const LinTile t = lin_tile(p, d->M, d->N);
    rc = lin_tile_check(t, p, a);
    if (rc) return rc;
    const Rows out{d->out, d->out_ld * es, (int64_t)d->N * es, d->M}, res{d->res, d->res_ld * es, (int64_t)d->N * es, d->M}, x{d->x, d->x_ld * es, (int64_t)d->K * es, d->M};
    const Rows xc{d->x ? nullptr : d->x_codes, d->xc_ld, p.nb * E2M1::BYTES, d->M}, xs{d->x ? nullptr : d->x_scales, d->xs_ld, p.nb, d->M};
    if (meet(out, x) || meet(out, xc) || meet(out, xs) || meet(out, {d->w, d->w_ld, p.nb * E2M1::BYTES, d->N}) || meet(out, {d->w_scales, d->s_ld, p.nb, d->N}))
        return msc_fail(MSC_ERR_ARG, "msc_mx_linear: out shares memory with x or w: other channels' blocks still read them");
    if (d->res != d->out && meet(out, res)) return msc_fail(MSC_ERR_ARG, "msc_mx_linear: out shares memory with res and is not res itself");
    // (nothing has been launched so far)
    if (p.pack) {
        rc = msc_mx_pack(d->x, d->x_ld, d->dtype, codes, p.xc_ld, scales, p.s_ld, MSC_MX_E2M1, d->M, d->K, stream);
        if (rc) return rc;
    }
    auto aligned_rows = [&](const uint8_t* s, long ld, int64_t rows, uint8_t* to) {
        hipLaunchKernelGGL(mx_scale_rows_kernel, dim3((unsigned)(rows < 4096 ? (rows + 3) / 4 : 1024)), dim3(256), 0, (hipStream_t)stream, s, ld, to, (long)p.s_ld, (long)rows, (int)p.nb);
    };
    if (p.scales && !p.pack) aligned_rows(d->x_scales, d->xs_ld, d->M, scales);
    if (p.w_scales) aligned_rows(d->w_scales, d->s_ld, d->N, w_scales);
    hipStream_t st = (hipStream_t)stream;
    rc = d->dtype == MSC_F32 ? lin_by_tile<float>(a, p, t, d, st) : d->dtype == MSC_BF16 ? lin_by_tile<bf16_t>(a, p, t, d, st) : lin_by_tile<f16_t>(a, p, t, d, st);
    return rc ? rc : msc_check_launch("msc_mx_linear");
}
