// Device helpers of the microscaled kernels (mx.hip, mx_wgrad.hip, mx_linear.hip): the block format of include/msc.h.
//
// Scale of a block.  With amax's float bits (E = exponent field, m = mantissa field) the smallest power of two s under which amax / s does not pass the
// largest code, top = 1.75 * 2^8 (E4M3) or 1.5 * 2^2 (E2M1), has the exponent field  E - 8 + [m > 0.75 * 2^23]  or  E - 2 + [m > 0.5 * 2^23]: integer
// operations on the bits, exact for every input.  Division by s is a product with the power of two of field 254 - e: exact (what would leave the
// normal range is far below the smallest code).  The conversions then round to nearest even once.
#pragma once
#include "common.h"

namespace mx {

constexpr int BLOCK = 32, MIN_E = 10, NAN_E = 255;

struct E4M3 {
    static constexpr int ID = 0, TOP = 8, BYTES = 32;                 // bytes per block
    static constexpr unsigned PAST = 0x600000u;
};
struct E2M1 {
    static constexpr int ID = 1, TOP = 2, BYTES = 16;
    static constexpr unsigned PAST = 0x400000u;
};
// largest magnitude kept (see the format's text): 1.875 / 1.5 times the type's largest power of two
template <typename F, typename T> __device__ __forceinline__ float limit() {
    const float top = F::ID == 0 ? 1.875f : 1.5f;
    return sizeof(T) == 2 && !__is_same(T, bf16_t) ? top * 32768.f : top * 0x1p127f;
}
template <typename F> __device__ __forceinline__ unsigned scale_field(unsigned amax_bits) {
    const int e = (int)(amax_bits >> 23) - F::TOP + ((amax_bits & 0x7fffffu) > F::PAST ? 1 : 0);
    return (unsigned)max(e, MIN_E);                                   // at most 255 - 2 + 1 = 254
}
__device__ __forceinline__ float pow2_field(unsigned e) { return __uint_as_float(e << 23); }
// 2^(e - 127) of a stored scale byte; NaN for 255.  Byte 0 is 2^-127, a denormal float whose one bit lies below the exponent field
__device__ __forceinline__ float scale_value(unsigned e) { return e == NAN_E ? __uint_as_float(0x7fc00000u) : __uint_as_float(max(e << 23, 0x400000u)); }
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 8 elements in units of the scale -> codes
__device__ __forceinline__ uint2 encode8_e4m3(const float* q) {
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    return make_uint2((unsigned)lo, (unsigned)hi);
}
__device__ __forceinline__ unsigned encode8_e2m1(const float* q) {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, q[0], q[1], 1.f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, q[2], q[3], 1.f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, q[4], q[5], 1.f, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, q[6], q[7], 1.f, 3);
    return r;
}
// 4 codes of a dword -> values times s
__device__ __forceinline__ void decode4_e4m3(unsigned w, float s, float* v) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a[0] * s; v[1] = a[1] * s; v[2] = b[0] * s; v[3] = b[1] * s;
}
__device__ __forceinline__ void decode8_e2m1(unsigned w, float s, float* v) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
    const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
    v[0] = a[0] * s; v[1] = a[1] * s; v[2] = b[0] * s; v[3] = b[1] * s;
    v[4] = c[0] * s; v[5] = c[1] * s; v[6] = d[0] * s; v[7] = d[1] * s;
}

// maximum over the four lanes of a quad (two DPP quad permutes); every lane of the quad is active
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));       // quad_perm [1,0,3,2]
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));       // quad_perm [2,3,0,1]
    return v;
}

// n / d for n < 2^31 by a multiplication: m = ceil(2^(31 + l) / d), l = ceil(log2 d) (Granlund and Montgomery, "Division by invariant integers
// using multiplication"); m < 2^32, and the error term is below 2^-31 * n / d < 1 / d
struct FastDiv {
    unsigned d, m, s;
};
static inline FastDiv fast_div(unsigned d) {
    unsigned l = 0;
    while ((1ull << l) < d) ++l;
    FastDiv f;
    f.d = d;
    f.m = (unsigned)(((1ull << (31 + l)) + d - 1) / d);
    f.s = l;
    return f;
}
__device__ __forceinline__ unsigned div_of(unsigned n, const FastDiv& f) { return (unsigned)(((unsigned long long)n * f.m) >> 31 >> f.s); }

// 8 consecutive elements of a row as floats: 16-byte loads, or one element at a time below `left` of them (the others zero)
// Elements of a row as they are stored, 16 bytes a unit, eight elements a chunk.  Whole units move at any alignment of their elements (the hardware's global
// accesses take it), so that odd widths and channel slices need no kernels of their own; the last unit of a row comes element by element, every
// load issued before the first is waited for.  Kept raw until they are used: converted at once, each load would be waited for before the next one goes out.
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2), may_alias));
template <typename T> __device__ __forceinline__ uint4 load_unit(const T* p, int left) {
    constexpr int N = Vec16<T>::N;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (left >= N) {
        v = __builtin_bit_cast(uint4, *reinterpret_cast<const u32x4_any*>(p));
    } else if (left > 0) {
        unsigned e[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(T) == 2) e[i] = *reinterpret_cast<const uint16_t*>(p + min(i, left - 1));
            else e[i] = *reinterpret_cast<const unsigned*>(p + min(i, left - 1));
        }
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = i < left ? e[i] : 0u;
        if constexpr (sizeof(T) == 2) v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        else v = make_uint4(e[0], e[1], e[2], e[3]);
    }
    return v;
}
template <typename T> struct Chunk {
    static constexpr int UNITS = sizeof(T) / 2;
    uint4 v[UNITS];
    __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
        for (int k = 0; k < UNITS; ++k) Vec16<T>::unpack(v[k], f + k * Vec16<T>::N);
    }
};
template <typename T> __device__ __forceinline__ Chunk<T> load_chunk(const T* p, int left) {
    Chunk<T> c;
#pragma unroll
    for (int k = 0; k < c.UNITS; ++k) c.v[k] = load_unit<T>(p + k * Vec16<T>::N, left - k * Vec16<T>::N);
    return c;
}
template <typename T> __device__ __forceinline__ void store_chunk(T* p, int left, const float* v) {
    constexpr int N = Vec16<T>::N;
    if (left >= 8) {
#pragma unroll
        for (int k = 0; k < 8 / N; ++k) *reinterpret_cast<u32x4_any*>(p + k * N) = __builtin_bit_cast(u32x4_any, Vec16<T>::pack(v + k * N));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) ElemIO<T>::store(p + i, v[i]);
    }
}

// one quad's block of 32: `v` the 8 elements of this lane, raw.  Returns the scale byte; q = the elements in units of the scale, zeros in a NaN block
template <typename F, typename T> __device__ __forceinline__ unsigned block_scale(const float* v, float* q) {
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, abs_bits(v[i]));
    a = quad_max(a);
    const float lim = limit<F, T>();
    const bool nan = a >= 0x7f800000u;
    const unsigned e = nan ? (unsigned)NAN_E : scale_field<F>(min(a, __float_as_uint(lim)));
    const float inv = nan ? 0.f : pow2_field(254 - e);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = nan ? 0.f : fminf(fmaxf(v[i], -lim), lim) * inv;
    return e;
}

// host: what every descriptor's packed operand has to satisfy
static inline bool packed_ok(const void* codes, int64_t ld, const void* scales, int64_t s_ld, int C, int block_bytes) {
    const int64_t nb = ((int64_t)C + BLOCK - 1) / BLOCK;
    return codes && scales && ((uintptr_t)codes & 15) == 0 && ld % 16 == 0 && ld >= nb * block_bytes && s_ld >= nb;
}
// Rows of `len` bytes, `pitch` bytes apart.  Two such sets of one pitch (channel slices of one buffer) share a byte where their columns do; of two pitches
// they are taken to share one as soon as the memory they span does.  Kernels write results while other blocks still read operands, so nothing but the in-place forms
// that a descriptor names may meet.
struct Rows { const void* p; int64_t pitch, len, rows; };
static inline bool meet(const Rows& a, const Rows& b) {
    if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0) return false;
    const __int128 a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p, a1 = a0 + (__int128)(a.rows - 1) * a.pitch + a.len, b1 = b0 + (__int128)(b.rows - 1) * b.pitch + b.len;
    if (a1 <= b0 || b1 <= a0) return false;
    const int64_t pitch = a.rows == 1 ? b.pitch : a.pitch;
    if ((a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) || (a.rows == 1 && b.rows == 1)) return true;
    const int64_t off = (int64_t)(((b0 - a0) % pitch + pitch) % pitch);
    return off < a.len || off + b.len > pitch;
}
static inline Rows one_row(const void* p, int64_t len) { return {p, len, len, 1}; }
static inline bool vec_ok(const void* p, int64_t ld, int dtype) { return ((uintptr_t)p & 15) == 0 && ld % msc_dtype_vec(dtype) == 0; }

}  // namespace mx
