// F8: 8-bit floating point with one scale per block of 128 - the quantiser and the matrix product (include/stylemesh_hip.h
// section F8). The reference computes in fp32 throughout and has no counterpart; the format is the next rung below this
// library's fp16x2 arithmetic (conv_split_kernel.h) and keeps its idea: operands scaled by powers of two.
//
//   x[r][c] = code[r][c] * 2^(s - 127)   codes e4m3 (largest 448) or e5m2 (57344), s = one byte per 128 columns of a row
//                                        ("rows") or per 128 x 128 tile ("tiles")
//   product: out[m][n] = sum_kb sa[m][kb] sb[n or n / 128][kb] sum_{k in block kb} a[m][k] b[n][k], fp32 accumulate
//
// Power-of-two scales make the quantiser exact up to the one rounding to 8 bits (x 2^-e is exact) and cost the product no
// instruction: they are part of the conversion that widens the codes to bf16, and for sums of fewer bits, where the caller permits
// them, v_mfma_scale_f32_16x16x128_f8f6f4 takes a block of 128 per instruction and one scale byte per operand row. fp32
// scales (any value) take the same kernels with the block's partial sum multiplied in on the vector unit.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace sm {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// loads / stores of memory that is aligned to its elements only
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));

__device__ __forceinline__ float bf16_to_f32(unsigned h) { return __builtin_bit_cast(float, h << 16); }
// round to nearest even; NaN stays NaN (its payload's top bit is set, or the carry could run into infinity)
__device__ __forceinline__ unsigned f32_to_bf16(float f) {
    const unsigned u = __builtin_bit_cast(unsigned, f);
    const unsigned r = (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
    return (u & 0x7fffffffu) > 0x7f800000u ? ((u >> 16) | 0x40u) : r;
}
__device__ __forceinline__ float f16_to_f32(unsigned h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }
__device__ __forceinline__ unsigned f32_to_f16(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

// 16 bytes of fp32 / bf16 / fp16 -> 4 / 8 floats
template <int T>
__device__ __forceinline__ void unpack(u32x4 a, float* v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (T == SM_TYPE_F32) v[j] = __builtin_bit_cast(float, (unsigned)a[j]);
        else {
            v[2 * j] = T == SM_TYPE_BF16 ? bf16_to_f32(a[j] & 0xffffu) : f16_to_f32(a[j] & 0xffffu);
            v[2 * j + 1] = T == SM_TYPE_BF16 ? __builtin_bit_cast(float, (unsigned)a[j] & 0xffff0000u) : f16_to_f32(a[j] >> 16);
        }
    }
}
// eight consecutive elements of a row as fp32 (type: SM_TYPE_*); `valid` of them exist, the others are 0
template <int T>
__device__ __forceinline__ void load8(const void* base, size_t off, int valid, float* v) {
    if (valid >= 8) {
        if constexpr (T == SM_TYPE_F32) {
            const u32x4_u* p = reinterpret_cast<const u32x4_u*>(static_cast<const float*>(base) + off);
            unpack<T>(p[0], v);
            unpack<T>(p[1], v + 4);
        } else {
            unpack<T>(*reinterpret_cast<const u32x4_u*>(static_cast<const uint16_t*>(base) + off), v);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = 0.f;
        if (j < valid) {
            if constexpr (T == SM_TYPE_F32) v[j] = static_cast<const float*>(base)[off + j];
            else {
                const unsigned h = static_cast<const uint16_t*>(base)[off + j];
                v[j] = T == SM_TYPE_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
            }
        }
    }
}

// |x| where it takes part in a block's maximum: infinities and NaN do not (they become NaN / infinity codes of their own and
// leave their neighbours' scale alone)
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.4028235e38f ? a : 0.f;
}

// The exponent e of a block's scale: the smallest with amax <= 1.75 * 2^top * 2^e (top = 8: e4m3, 15: e5m2), read off the
// bits of amax (a subnormal one is normalised first); clamped to [-127, 127]. amax = 0 -> 0.
__device__ __forceinline__ int block_exponent(float amax, int top) {
    unsigned u = __builtin_bit_cast(unsigned, amax);
    if (u == 0) return 0;
    int ex = (int)(u >> 23);
    unsigned man = u & 0x7fffffu;
    if (ex == 0) {
        const int z = __builtin_clz(man) - 8;      // leading zeros in front of the 24-bit significand
        man = (man << z) & 0x7fffffu;
        ex = 1 - z;
    }
    const int e = ex - 127 - top + (man > 0x600000u ? 1 : 0);   // significand > 1.75
    return max(-127, min(127, e));
}
// 2^-e for e in [-127, 127]
__device__ __forceinline__ float inv_pow2(int e) {
    return e == 127 ? __builtin_bit_cast(float, 0x00400000u) : __builtin_bit_cast(float, (unsigned)(127 - e) << 23);
}

// two scaled values -> two codes in the low (HI = false) or high half of `old`. Scaled finite values are within the format's
// range by construction of the scale, so no saturation takes place; e4m3 has no infinity: it becomes NaN like a NaN does.
template <bool HI>
__device__ __forceinline__ int cvt2(float a, float b, int old, int fmt) {
    if (fmt == SM_FP8_E4M3) {
        const float qn = __builtin_bit_cast(float, 0x7fc00000u);
        a = fabsf(a) <= 448.f ? a : qn;
        b = fabsf(b) <= 448.f ? b : qn;
        return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, HI);
    }
    return __builtin_amdgcn_cvt_pk_bf8_f32(a, b, old, HI);
}
__device__ __forceinline__ u32x2 cvt8(const float* v, float inv, int fmt) {
    u32x2 r;
    int w = cvt2<false>(v[0] * inv, v[1] * inv, 0, fmt);
    r[0] = (unsigned)cvt2<true>(v[2] * inv, v[3] * inv, w, fmt);
    w = cvt2<false>(v[4] * inv, v[5] * inv, 0, fmt);
    r[1] = (unsigned)cvt2<true>(v[6] * inv, v[7] * inv, w, fmt);
    return r;
}

// Where the scale byte of (row, block kb) lives: [kb / 4][row][kb % 4] - the four bytes of a dword are the four blocks the
// product's matrix instructions pick from one register (op_sel).
__device__ __forceinline__ size_t scale_at(int kb, int row, int rows) { return ((size_t)(kb >> 2) * rows + row) * 4 + (kb & 3); }

struct QuantArgs {
    const void* x;
    size_t stride;
    int rows, cols, fmt;
    uint8_t *q, *qs, *qt, *qts;
};

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Magnitudes compare like their bits: a dword holds one fp32 or two 16-bit ones, and maxima are integer maxima.
template <int T>
__device__ __forceinline__ unsigned mag(unsigned d) { return d & (T == SM_TYPE_F32 ? 0x7fffffffu : 0x7fff7fffu); }
template <int T>
__device__ __forceinline__ unsigned mag_max(unsigned a, unsigned b) {
    if constexpr (T == SM_TYPE_F32) return max(a, b);
    else return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <int T>
constexpr unsigned inf_bits = T == SM_TYPE_F32 ? 0x7f800000u : T == SM_TYPE_BF16 ? 0x7f80u : 0x7c00u;
template <int T>
__device__ __forceinline__ unsigned mag_both(unsigned m) { return T == SM_TYPE_F32 ? m : max(m & 0xffffu, m >> 16); }   // of a dword's values
template <int T>
__device__ __forceinline__ unsigned mag_finite(unsigned m) {      // non-finite values -> 0
    if constexpr (T == SM_TYPE_F32) return m >= inf_bits<T> ? 0u : m;
    else return ((m & 0xffffu) >= inf_bits<T> ? 0u : m & 0xffffu) | ((m >> 16) >= inf_bits<T> ? 0u : m & 0xffff0000u);
}
template <int T>
__device__ __forceinline__ float mag_float(unsigned m) {
    return T == SM_TYPE_F32 ? __builtin_bit_cast(float, m) : T == SM_TYPE_BF16 ? bf16_to_f32(m) : f16_to_f32(m);
}
// max over the 16 lanes of a row of the wave (data-parallel moves, no LDS)
template <int T>
__device__ __forceinline__ unsigned row16_max(unsigned m) {
    m = mag_max<T>(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, false));      // row_ror 8, 4, 2, 1
    m = mag_max<T>(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, false));
    m = mag_max<T>(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, false));
    return mag_max<T>(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, false));
}

// Two finite values divided by 2^e -> two codes: one instruction, round to nearest even (scale: the float 2^e, normal).
// 16-bit types: v = the dword of both; fp32: v and w.
template <int T, bool HI>
__device__ __forceinline__ s16x2 cvt_scaled(unsigned v, unsigned w, float scale, s16x2 old, int fmt) {
    if (fmt == SM_FP8_E4M3) {
        if constexpr (T == SM_TYPE_F32) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(old, __builtin_bit_cast(float, v), __builtin_bit_cast(float, w), scale, HI);
        else if constexpr (T == SM_TYPE_BF16) return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, __builtin_bit_cast(bf16x2, v), scale, HI);
        else return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, __builtin_bit_cast(f16x2, v), scale, HI);
    }
    if constexpr (T == SM_TYPE_F32) return __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(old, __builtin_bit_cast(float, v), __builtin_bit_cast(float, w), scale, HI);
    else if constexpr (T == SM_TYPE_BF16) return __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(old, __builtin_bit_cast(bf16x2, v), scale, HI);
    else return __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(old, __builtin_bit_cast(f16x2, v), scale, HI);
}
// N values (four or eight) of a row (16-bit: N / 2 dwords, fp32: N) -> N codes. plain: all finite and the scale a normal float;
// otherwise each value is scaled and selected on its own.
template <int T, int N>
struct Codes {
    unsigned w[N / 4];
};
template <int T, int N>
__device__ __forceinline__ Codes<T, N> encode(const unsigned* d, int e, int fmt, bool plain) {
    Codes<T, N> r;
    if (plain) {
        const float scale = __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
#pragma unroll
        for (int h = 0; h < N / 4; ++h) {
            s16x2 c = {0, 0};
            if constexpr (T == SM_TYPE_F32) {
                c = cvt_scaled<T, false>(d[4 * h], d[4 * h + 1], scale, c, fmt);
                c = cvt_scaled<T, true>(d[4 * h + 2], d[4 * h + 3], scale, c, fmt);
            } else {
                c = cvt_scaled<T, false>(d[2 * h], 0, scale, c, fmt);
                c = cvt_scaled<T, true>(d[2 * h + 1], 0, scale, c, fmt);
            }
            r.w[h] = __builtin_bit_cast(unsigned, c);
        }
        return r;
    }
    const float inv = inv_pow2(e);
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
        float v[8];
        if constexpr (T == SM_TYPE_F32) unpack<T>(u32x4{d[4 * h], d[4 * h + 1], d[4 * h + 2], d[4 * h + 3]}, v);
        else unpack<T>(u32x4{d[2 * h], d[2 * h + 1], 0u, 0u}, v);
        const int w = cvt2<false>(v[0] * inv, v[1] * inv, 0, fmt);
        r.w[h] = (unsigned)cvt2<true>(v[2] * inv, v[3] * inv, w, fmt);
    }
    return r;
}
template <int T>
__device__ __forceinline__ u32x2 codes8(const unsigned* d, int e, int fmt, bool plain) {
    const Codes<T, 8> c = encode<T, 8>(d, e, fmt, plain);
    return u32x2{c.w[0], c.w[1]};
}

// columns c0 ... c0 + 7 of rows r0 ... r0 + RPT - 1 as they are, all loads in flight together; zeros outside the matrix
template <int T, int RPT, int ND>
__device__ __forceinline__ void load_rows(const QuantArgs& a, int r0, int c0, unsigned (&d)[RPT][ND]) {
    constexpr int ES = T == SM_TYPE_F32 ? 4 : 2;
    if (c0 + 8 <= a.cols) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = min(r0 + i, a.rows - 1);
            const u32x4_u* p = reinterpret_cast<const u32x4_u*>(static_cast<const char*>(a.x) + ((size_t)r * a.stride + c0) * ES);
#pragma unroll
            for (int q = 0; q < ND / 4; ++q) {
                const u32x4 w = p[q];
#pragma unroll
                for (int j = 0; j < 4; ++j) d[i][4 * q + j] = w[j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = min(r0 + i, a.rows - 1);
#pragma unroll
            for (int j = 0; j < ND; ++j) {
                const size_t at = (size_t)r * a.stride + c0;
                if constexpr (T == SM_TYPE_F32) {
                    d[i][j] = c0 + j < a.cols ? static_cast<const unsigned*>(a.x)[at + j] : 0u;
                } else {
                    const uint16_t* p = static_cast<const uint16_t*>(a.x) + at;
                    d[i][j] = (c0 + 2 * j < a.cols ? (unsigned)p[2 * j] : 0u) | (c0 + 2 * j + 1 < a.cols ? (unsigned)p[2 * j + 1] << 16 : 0u);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i)
        if (r0 + i >= a.rows)
#pragma unroll
            for (int j = 0; j < ND; ++j) d[i][j] = 0;
}

// One tile of ROWS rows x 128 columns per block: thread t holds rows RPT (t / 16) ... and columns 8 (t % 16) ... + 7 as they came
// (all its loads in flight together; x is read once whatever is produced). Maxima are taken on the bits, two 16-bit
// values per instruction: a block row's 16 lanes by data-parallel moves; columns in registers, then the wave's four row
// groups, then the waves through LDS; tiles over everything. The scaled conversion instruction does the rest (about three
// instructions an element where it was twenty). The transposed codes turn through a 128 x 128 byte LDS image whose 8-byte units are
// swizzled by their column group, and both results leave as whole 128-byte lines.
// A column's exponent is found by one thread and read back by the sixteen that hold its rows (each on its own: 4096^2 bf16 both
// ways 19.7 -> 17.6 us, the LDS reads and integer instructions of it).
// Bound by HBM: rows * cols * (sizeof(x) + 1 per result); 8192^2 bf16 both ways 60 us, 4.5 TB/s (a copy of that size: 5.3).
// Transposes and tiles take ROWS = 128, RPT = 4: with few tiles a thread's instructions bound it (1029 x 517 fp32 both
// ways 9.1 us at RPT = 8, 7.2 at 4; no difference at 8192^2). Rows alone take RPT = 8, and 16 rows a block, RPT = 1, where
// 128 leave too few blocks (16 x 4096 fp32: 8.2 -> 2.7 us).
template <int T, bool TILES, bool Q, bool QT, int RPT, int ROWS>
__device__ __forceinline__ void quantize_tile(const QuantArgs& a, const int bx, const int by) {
    static_assert(ROWS == 128 || (!TILES && !QT), "column blocks need 128 rows");
    static_assert(!QT || RPT == 4, "a dword of a column per thread");
    constexpr int NT = 16 * ROWS / RPT, NW = NT / 64;
    constexpr int ND = T == SM_TYPE_F32 ? 8 : 4;      // dwords of eight values
    const int tid = threadIdx.x, rg = tid >> 4, cg = tid & 15, wave = tid >> 6;
    const int tr = by * ROWS, tc = bx * 128, c0 = tc + cg * 8;
    const int top = a.fmt == SM_FP8_E4M3 ? 8 : 15;
    unsigned d[RPT][ND];
    load_rows<T, RPT>(a, tr + rg * RPT, c0, d);
    unsigned rmax[RPT], all = 0;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < ND; ++j) m = mag_max<T>(m, mag<T>(d[i][j]));
        rmax[i] = m;
        all = mag_max<T>(all, m);
    }
    // a wave that holds infinities or NaN takes its maxima again without them, and converts value by value
    const bool finite = !__any(mag_both<T>(all) >= inf_bits<T>);
    if (!finite) {
        all = 0;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < ND; ++j) m = mag_max<T>(m, mag_finite<T>(mag<T>(d[i][j])));
            rmax[i] = m;
            all = mag_max<T>(all, m);
        }
    }
    __shared__ unsigned red[NW][QT && !TILES ? 16 * ND : 1];
    __shared__ __align__(16) uint8_t img[QT ? 128 * 128 : 16];
    __shared__ __align__(16) int exponent[QT && !TILES ? 128 : 4];
    const int cblocks = (a.cols + 127) >> 7, rblocks = (a.rows + 127) >> 7;
    int tile_e = 0;
    if constexpr (TILES) {
        unsigned m = mag_both<T>(all);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
        if ((tid & 63) == 0) red[wave][0] = m;
        __syncthreads();
        m = red[0][0];
#pragma unroll
        for (int w = 1; w < NW; ++w) m = max(m, red[w][0]);
        tile_e = block_exponent(mag_float<T>(m), top);
        if (tid < 4) {      // thread 0: this tile's byte; the row's / column's last tile also fills the dword's unused bytes
            if (Q && (tid == 0 || (bx + tid < (cblocks + 3) / 4 * 4 && bx == cblocks - 1)))
                a.qs[scale_at(bx + tid, by, rblocks)] = tid == 0 ? (uint8_t)(tile_e + 127) : (uint8_t)127;
            if (QT && (tid == 0 || (by + tid < (rblocks + 3) / 4 * 4 && by == rblocks - 1)))
                a.qts[scale_at(by + tid, bx, cblocks)] = tid == 0 ? (uint8_t)(tile_e + 127) : (uint8_t)127;
        }
    }
    if constexpr (Q) {
        const size_t pitch = (size_t)cblocks * 128;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = tr + rg * RPT + i;
            const int e = TILES ? tile_e : block_exponent(mag_float<T>(mag_both<T>(row16_max<T>(rmax[i]))), top);
            if (r < a.rows) {
                *reinterpret_cast<u32x2*>(a.q + (size_t)r * pitch + c0) = codes8<T>(d[i], e, a.fmt, finite && !__any(e == -127));
                if (!TILES && cg < 4 && (cg == 0 || (bx == cblocks - 1 && bx + cg < (cblocks + 3) / 4 * 4)))
                    a.qs[scale_at(bx + cg, r, a.rows)] = cg == 0 ? (uint8_t)(e + 127) : (uint8_t)127;
            }
        }
    }
    if constexpr (QT) {
        if constexpr (!TILES) {
#pragma unroll
            for (int j = 0; j < ND; ++j) {
                unsigned m = 0;
                if (finite) {
#pragma unroll
                    for (int i = 0; i < RPT; ++i) m = mag_max<T>(m, mag<T>(d[i][j]));
                } else {
#pragma unroll
                    for (int i = 0; i < RPT; ++i) m = mag_max<T>(m, mag_finite<T>(mag<T>(d[i][j])));
                }
                m = mag_max<T>(m, (unsigned)__shfl_xor((int)m, 16, 64));
                m = mag_max<T>(m, (unsigned)__shfl_xor((int)m, 32, 64));
                if ((tid & 63) < 16) red[wave][cg * ND + j] = m;
            }
            __syncthreads();
            if (tid < 128) {      // a thread per column
                unsigned m = 0;
#pragma unroll
                for (int w = 0; w < NW; ++w) m = mag_max<T>(m, red[w][T == SM_TYPE_F32 ? tid : tid >> 1]);
                if constexpr (T != SM_TYPE_F32) m = tid & 1 ? m >> 16 : m & 0xffffu;
                exponent[tid] = block_exponent(mag_float<T>(m), top);
                if (tc + tid < a.cols) {
                    a.qts[scale_at(by, tc + tid, a.cols)] = (uint8_t)(exponent[tid] + 127);
                    if (by == rblocks - 1)      // the dword's unused bytes
                        for (int k = rblocks; k & 3; ++k) a.qts[scale_at(k, tc + tid, a.cols)] = 127;
                }
            }
            __syncthreads();
        }
        int es[8];
        bool plain = finite;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            es[j] = TILES ? tile_e : exponent[cg * 8 + j];
            plain = plain && es[j] != -127;
        }
        plain = __all(plain);
#pragma unroll
        for (int j = 0; j < 8; ++j) {      // column j of the thread: its rows, packed as a row of the transpose
            const int cl = cg * 8 + j, dj = T == SM_TYPE_F32 ? j : j >> 1;
            constexpr int NR = T == SM_TYPE_F32 ? RPT : RPT / 2;
            unsigned t[NR];
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                if constexpr (T == SM_TYPE_F32) t[i] = d[i][j];
                else t[i] = j & 1 ? (d[2 * i][dj] >> 16) | (d[2 * i + 1][dj] & 0xffff0000u) : (d[2 * i][dj] & 0xffffu) | (d[2 * i + 1][dj] << 16);
            }
            *reinterpret_cast<unsigned*>(img + cl * 128 + ((rg >> 1) ^ cg) * 8 + (rg & 1) * 4) =
                encode<T, 4>(t, es[j], a.fmt, plain).w[0];
        }
        __syncthreads();
        const size_t pitch = (size_t)rblocks * 128;
#pragma unroll
        for (int i = 0; i < 1024 / NT; ++i) {      // 8 lanes write a column's 128 bytes
            const int cl = i * (NT / 8) + (tid >> 3), p = tid & 7, g = cl >> 3;
            // units 2 p and 2 p + 1 of the column lie in the pair p ^ (g / 2), the other way round for odd g
            u32x4 w = *reinterpret_cast<const u32x4*>(img + cl * 128 + (p ^ (g >> 1)) * 16);
            if (g & 1) w = u32x4{w[2], w[3], w[0], w[1]};
            if (tc + cl < a.cols) *reinterpret_cast<u32x4*>(a.qt + (size_t)(tc + cl) * pitch + tr + p * 16) = w;
        }
    }
}

template <int T, bool TILES, bool Q, bool QT, int RPT, int ROWS>
__global__ __launch_bounds__(16 * ROWS / RPT) void fp8_quantize_kernel(QuantArgs a) {
    quantize_tile<T, TILES, Q, QT, RPT, ROWS>(a, blockIdx.x, blockIdx.y);
}

// 128 rows x 32 columns of the transpose: thread t holds rows 2 (t / 4), + 1 and columns 8 (t % 4) ... + 7; as above otherwise. The
// image's 32-byte units are swizzled by the column group.
template <int T>
__device__ __forceinline__ void quantize_columns(const QuantArgs& a, const int bx, const int by) {
    constexpr int ND = T == SM_TYPE_F32 ? 8 : 4;
    const int tid = threadIdx.x, rg = tid >> 2, cg = tid & 3, wave = tid >> 6;
    const int tr = by * 128, tc = bx * 32;
    const int top = a.fmt == SM_FP8_E4M3 ? 8 : 15;
    const int rblocks = (a.rows + 127) >> 7;
    unsigned d[2][ND];
    load_rows<T, 2>(a, tr + rg * 2, tc + cg * 8, d);
    unsigned all = 0;
#pragma unroll
    for (int j = 0; j < ND; ++j) all = mag_max<T>(all, mag_max<T>(mag<T>(d[0][j]), mag<T>(d[1][j])));
    const bool finite = !__any(mag_both<T>(all) >= inf_bits<T>);
    __shared__ unsigned red[4][4 * ND];
    __shared__ __align__(16) int exponent[32];
    __shared__ __align__(16) uint8_t img[32 * 128];
#pragma unroll
    for (int j = 0; j < ND; ++j) {
        unsigned m = finite ? mag_max<T>(mag<T>(d[0][j]), mag<T>(d[1][j])) : mag_max<T>(mag_finite<T>(mag<T>(d[0][j])), mag_finite<T>(mag<T>(d[1][j])));
#pragma unroll
        for (int o = 4; o < 64; o <<= 1) m = mag_max<T>(m, (unsigned)__shfl_xor((int)m, o, 64));
        if ((tid & 63) < 4) red[wave][cg * ND + j] = m;
    }
    __syncthreads();
    if (tid < 32) {      // a thread per column
        const int dj = T == SM_TYPE_F32 ? tid : tid >> 1;
        unsigned m = mag_max<T>(mag_max<T>(red[0][dj], red[1][dj]), mag_max<T>(red[2][dj], red[3][dj]));
        if constexpr (T != SM_TYPE_F32) m = tid & 1 ? m >> 16 : m & 0xffffu;
        const int e = block_exponent(mag_float<T>(m), top);
        exponent[tid] = e;
        if (tc + tid < a.cols) {
            a.qts[scale_at(by, tc + tid, a.cols)] = (uint8_t)(e + 127);
            if (by == rblocks - 1)      // the dword's unused bytes
                for (int k = rblocks; k & 3; ++k) a.qts[scale_at(k, tc + tid, a.cols)] = 127;
        }
    }
    __syncthreads();
    int es[8];
    bool plain = finite;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        es[j] = exponent[cg * 8 + j];
        plain = plain && es[j] != -127;
    }
    plain = __all(plain);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int cl = cg * 8 + j, dj = T == SM_TYPE_F32 ? j : j >> 1, e = es[j];
        unsigned c;
        if (plain) {
            const float scale = __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
            unsigned v, w = 0;
            if constexpr (T == SM_TYPE_F32) v = d[0][j], w = d[1][j];
            else v = j & 1 ? (d[0][dj] >> 16) | (d[1][dj] & 0xffff0000u) : (d[0][dj] & 0xffffu) | (d[1][dj] << 16);
            c = __builtin_bit_cast(unsigned, cvt_scaled<T, false>(v, w, scale, s16x2{0, 0}, a.fmt));
        } else {
            float v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = mag_float<T>(T == SM_TYPE_F32 ? d[i][j] : j & 1 ? d[i][dj] >> 16 : d[i][dj] & 0xffffu);
            const float inv = inv_pow2(e);
            c = (unsigned)cvt2<false>(v[0] * inv, v[1] * inv, 0, a.fmt);
        }
        *reinterpret_cast<uint16_t*>(img + cl * 128 + ((rg * 2) ^ (cg * 32))) = (uint16_t)c;
    }
    __syncthreads();
    const int cl = tid >> 3, p = tid & 7;
    if (tc + cl < a.cols)
        *reinterpret_cast<u32x4*>(a.qt + (size_t)(tc + cl) * ((size_t)rblocks * 128) + tr + p * 16) =
            *reinterpret_cast<const u32x4*>(img + cl * 128 + ((p * 16) ^ ((cl >> 3) * 32)));
}

// A small matrix row-wise and / or transposed: the first blocks_q blocks take 16 rows x 128 columns of the row-wise result, the others
// 128 x 32 of the transpose. x is read twice, the second time from the caches.
template <int T>
__global__ __launch_bounds__(256) void fp8_quantize_small_kernel(QuantArgs a, int blocks_q) {
    const int b = blockIdx.x;
    if (b < blocks_q) {
        const int cblocks = (a.cols + 127) >> 7;
        quantize_tile<T, false, true, false, 1, 16>(a, b % cblocks, b / cblocks);
    } else {
        const int ct = (a.cols + 31) >> 5, t = b - blocks_q;
        quantize_columns<T>(a, t % ct, t / ct);
    }
}

// ---- the product ---------------------------------------------------------------------------------------------------
struct MatmulArgs {
    const uint8_t* a;       // [M][a_pitch] codes
    const uint8_t* b;       // [N][b_pitch]
    const void* as;         // scales of a: bytes [KB / 4][M][4] or floats [KB][M]
    const void* bs;         // of b, rows M -> N (rows) or N / 128 (tiles)
    void* out;
    float* ws;              // split K: slabs [split][M][N]
    size_t a_pitch, b_pitch, out_stride;
    int M, N, KB;           // KB = blocks of 128 along K
    int b_shift;            // 0: b's scales per row, 7: per 128 rows
    int bs_rows;
    int out_type, accumulate;
    int kb_per_split;
};

// four results of a row in one store (results start at any element: aligned to theirs only); fewer at the row's end
__device__ __forceinline__ void store4(const MatmulArgs& g, int m, int n, f32x4 v) {
    const int cnt = g.N - n;
    const size_t at = (size_t)m * g.out_stride + n;
    if (g.out_type == SM_TYPE_F32) {
        float* o = static_cast<float*>(g.out) + at;
        if (cnt >= 4) {
            if (g.accumulate) {
                const u32x4 old = *reinterpret_cast<const u32x4_u*>(o);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += __builtin_bit_cast(float, (unsigned)old[j]);
            }
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(unsigned, (float)v[j]);
            *reinterpret_cast<u32x4_u*>(o) = w;
            return;
        }
        for (int j = 0; j < cnt; ++j) o[j] = g.accumulate ? o[j] + v[j] : v[j];
    } else {
        uint16_t* o = static_cast<uint16_t*>(g.out) + at;
        const bool bf = g.out_type == SM_TYPE_BF16;
        if (cnt >= 4) {
            if (g.accumulate) {
                const u32x2 old = *reinterpret_cast<const u32x2_u*>(o);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned h = (old[j >> 1] >> (16 * (j & 1))) & 0xffffu;
                    v[j] += bf ? bf16_to_f32(h) : f16_to_f32(h);
                }
            }
            u32x2 w;
            w[0] = bf ? f32_to_bf16(v[0]) | (f32_to_bf16(v[1]) << 16) : f32_to_f16(v[0]) | (f32_to_f16(v[1]) << 16);
            w[1] = bf ? f32_to_bf16(v[2]) | (f32_to_bf16(v[3]) << 16) : f32_to_f16(v[2]) | (f32_to_f16(v[3]) << 16);
            *reinterpret_cast<u32x2_u*>(o) = w;
            return;
        }
        for (int j = 0; j < cnt; ++j) {
            float x = v[j];
            if (g.accumulate) x += bf ? bf16_to_f32(o[j]) : f16_to_f32(o[j]);
            o[j] = (uint16_t)(bf ? f32_to_bf16(x) : f32_to_f16(x));
        }
    }
}

// Direct loads into LDS are counted as vector-memory operations and finish in their order. The waves of a block meet with
// their own loads - all but the LEFT newest - landed and their LDS reads done: after it every wave may read the stage
// those loads filled and overwrite the one those reads came from. (__syncthreads would wait for every load in flight.)
template <int LEFT>
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// An operand's 32 codes of a lane as bf16, scaled by 2^(byte - 127): e4m3 / e5m2 have 4 / 3 significant bits, bf16 has 8 and
// fp32's exponents, so this is exact where bf16 holds code 2^(byte - 127) as a normal number: bytes 32 ... 223 do for every code (17
// ... 239 of e5m2, 10 ... 246 of e4m3). Beyond them the scale is applied to the block's sum. scale: the byte in the
// exponent field of a float.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct Wide {
    bf16x8 p[4];
};
__device__ __forceinline__ i32x8 join(u32x4 lo, u32x4 hi) {
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
template <int F>
__device__ __forceinline__ Wide widen(i32x8 v, float scale) {
    Wide w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bf16x2 lo, hi;
        if constexpr (F == SM_FP8_E4M3) {
            lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[i], scale, false);
            hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[i], scale, true);
        } else {
            lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((unsigned)v[i], scale, false);
            hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((unsigned)v[i], scale, true);
        }
        w.p[i >> 1][(i & 1) * 4 + 0] = lo[0];
        w.p[i >> 1][(i & 1) * 4 + 1] = lo[1];
        w.p[i >> 1][(i & 1) * 4 + 2] = hi[0];
        w.p[i >> 1][(i & 1) * 4 + 3] = hi[1];
    }
    return w;
}
template <int OP>
__device__ __forceinline__ float byte_scale(int dword) {      // byte OP of a scale dword, 2^(byte - 127)
    const unsigned u = (unsigned)dword >> (8 * OP);
    return __builtin_bit_cast(float, (u & 255u) << 23);
}
// fp32 scales of a block meet its sum c, |c| in 2^-25 ... 2^32 or 0, as (c sa) sb, which leaves fp32's normal range before the
// result does only where sa other than 0 is outside 2^-95 ... 2^88 (1e20 x 1e20 over a small sum, or a zero one, is fine), or, where
// one sb serves many elements, as c (sa sb): there sa and sb have to lie in 2^-62 ... 2^63. Elsewhere significands and exponents
// are multiplied apart, and only the whole product is rounded into fp32's range.
struct ScaleRange {
    unsigned hi = 0, lo = ~0u;
    __device__ __forceinline__ void take(unsigned bits) {
        hi = max(hi, bits << 1);
        lo = min(lo, (bits << 1) - 1u);      // (0 is neither large nor small)
    }
    __device__ __forceinline__ bool far(bool both) const {
        return hi >= (both ? 190u : 215u) << 24 || lo < ((both ? 65u : 32u) << 24) - 1u;
    }
};
__device__ __forceinline__ float apart(float c, float sa, float sb) {
    return __builtin_amdgcn_ldexpf(c * (__builtin_amdgcn_frexp_mantf(sa) * __builtin_amdgcn_frexp_mantf(sb)),
                                   __builtin_amdgcn_frexp_expf(sa) + __builtin_amdgcn_frexp_expf(sb));
}
// the top bit of every byte of d that is in 32 ... 223 (its three top bits are not alike)
__device__ __forceinline__ unsigned bytes_near(unsigned d) { return (d ^ (d << 1)) | (d ^ (d << 2)); }
// c 2^(a - 127) 2^(b - 127), rounded once
__device__ __forceinline__ float apart(float c, int a, int b) {
    return a == 255 || b == 255 ? __builtin_bit_cast(float, 0x7fc00000u) : __builtin_amdgcn_ldexpf(c, a + b - 254);
}
// c[i] += b[i] a over a block of 128 for N rows of tiles: the four instructions of one result depend on each other, so the
// tiles take turns
template <int N>
__device__ __forceinline__ void mfma_wide(const Wide* b, const Wide& a, f32x4* c) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[i].p[q], a.p[q], c[i], 0, 0, 0);
}

template <int OP, int FA>
__device__ __forceinline__ f32x4 mfma_block(i32x8 bfrag, i32x8 afrag, f32x4 c, int sb, int sa) {
    // first operand = rows of b (the result's rows), second = rows of a: a lane ends up with four consecutive n of one m
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bfrag, afrag, c, SM_FP8_E4M3, FA, OP, sb, OP, sa);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)0xfffffff0u, 0x00020000);
}

// 16 bytes per lane from rsrc + voff + soff to LDS bytes dst + 16 lane (the builtin exists in the device pass only)
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, uint8_t* dst, unsigned voff, int soff) {
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)dst, 16, (int)voff, soff, 0, 0);
#endif
}

// BM x BN output tile per block, waves WM x WN; a stage = one block of 128 along K of both operands, in a ring of NST
// stages in LDS, filled by direct loads (16 bytes per lane, no registers). LDS rows are 128 bytes; the 16-byte chunk c of row r
// sits at chunk c ^ (r & 7), so that the eight lanes of a read phase hit eight different chunk columns. A lane's 32 bytes of
// an operand row are chunks g and g + 4 (g = lane / 16): the same permutation of k on both sides leaves the sum as it is,
// and a block of 128 has ONE scale, so it does not matter which quarter a lane holds.
enum { SCALE_POW2, SCALE_F32_ROWS, SCALE_F32_TILES };      // how the scales of a launch are held (fp32: B's blocks)

template <int BM, int BN, int WM, int WN, int NST, int FA, int SC, bool NATIVE>
__device__ __forceinline__ void matmul_tile(const MatmulArgs& g, int block) {
    constexpr int NT = WM * WN * 64;
    constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    __shared__ __align__(16) uint8_t lds[NST][(BM + BN) * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const int mt = (g.M + BM - 1) / BM, nt = (g.N + BN - 1) / BN;
    // XCD-contiguous shares of the tiles, walked in groups of 8 rows of tiles: the blocks of an XCD share operand rows in its L2
    const int id = xcd_linear(block, mt * nt);
    const int group = id / (8 * nt), gm = min(8, mt - group * 8), in = id - group * 8 * nt;
    const int m0 = (group * 8 + in % gm) * BM, n0 = in / gm * BN;
    const int kb0 = blockIdx.y * g.kb_per_split, kb1 = min(g.KB, kb0 + g.kb_per_split);

    // One direct load moves 64 lanes x 16 bytes = 8 rows; lane i's data lands at byte 16 i of the wave's kilobyte. Buffer loads: a
    // uniform base (the tile's first row), a 32-bit offset per lane (256 rows of the longest pitch stay below 2^32) and the
    // block of 128 as scalar offset - no 64-bit vector arithmetic in the loop. Rows behind the last are the last one again.
    constexpr int RW = NT / 8;                                   // rows all waves load at a time
    constexpr int NLA = BM / RW, NLB = BN / RW;
    static_assert(BM % RW == 0 && BN % RW == 0, "whole loads");
    const int r8 = lane >> 3, c16 = ((lane & 7) ^ r8) << 4;
    const __amdgpu_buffer_rsrc_t asrc = tile_rsrc(g.a + (size_t)m0 * g.a_pitch), bsrc = tile_rsrc(g.b + (size_t)n0 * g.b_pitch);
    unsigned va[NLA], vb[NLB];
#pragma unroll
    for (int i = 0; i < NLA; ++i) va[i] = (unsigned)min(i * RW + wave * 8 + r8, g.M - 1 - m0) * (unsigned)g.a_pitch + c16;
#pragma unroll
    for (int i = 0; i < NLB; ++i) vb[i] = (unsigned)min(i * RW + wave * 8 + r8, g.N - 1 - n0) * (unsigned)g.b_pitch + c16;
    auto stage = [&](int buf, int kb) {
        uint8_t* dst = lds[buf] + wave * 1024;
#pragma unroll
        for (int i = 0; i < NLA; ++i)
            load_to_lds(asrc, dst + i * RW * 128, va[i], kb * 128);
#pragma unroll
        for (int i = 0; i < NLB; ++i)
            load_to_lds(bsrc, dst + BM * 128 + i * RW * 128, vb[i], kb * 128);
    };
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int lr = lane & 15, lg = lane >> 4;
    // The scales of the next four blocks (power-of-two: a dword per row) or the next block (fp32) are loaded a step ahead.
    // rows of A: one per lane and row tile; rows of B: likewise, or - fp32, whose factors meet the result - the lane's four
    // result columns; fp32 scales per tile: one for the wave (its columns lie within one tile).
    constexpr bool F32S = SC != SCALE_POW2;
    constexpr int NB = SC == SCALE_POW2 ? TN : SC == SCALE_F32_ROWS ? 4 * TN : 1;
    unsigned arow[TM], brow[NB];
#pragma unroll
    for (int j = 0; j < TM; ++j) arow[j] = (unsigned)min(m0 + (wm * TM + j) * 16 + lr, g.M - 1) * 4u;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int n = n0 + wn * TN * 16 + (SC == SCALE_POW2 ? i * 16 + lr : SC == SCALE_F32_ROWS ? (i >> 2) * 16 + lg * 4 + (i & 3) : 0);
        brow[i] = (unsigned)(min(n, g.N - 1) >> g.b_shift) * 4u;
    }
    int sa[TM], sb[NB], sa_next[TM], sb_next[NB];
    auto load_scales = [&](int row, int* pa_out, int* pb_out) {      // row: of the scale arrays (kb / 4 or kb)
        const __amdgpu_buffer_rsrc_t pa = tile_rsrc(static_cast<const char*>(g.as) + (size_t)row * g.M * 4);
        const __amdgpu_buffer_rsrc_t pb = tile_rsrc(static_cast<const char*>(g.bs) + (size_t)row * g.bs_rows * 4);
#pragma unroll
        for (int j = 0; j < TM; ++j) pa_out[j] = (int)__builtin_amdgcn_raw_buffer_load_b32(pa, arow[j], 0, 0);
#pragma unroll
        for (int i = 0; i < NB; ++i) pb_out[i] = (int)__builtin_amdgcn_raw_buffer_load_b32(pb, brow[i], 0, 0);
    };
    auto take_scales = [&]() {
#pragma unroll
        for (int j = 0; j < TM; ++j) sa[j] = sa_next[j];
#pragma unroll
        for (int i = 0; i < NB; ++i) sb[i] = sb_next[i];
    };
    // a tile of 16 rows is 2 KB of LDS; the swizzle depends on the row within it only
    const int f0 = lr * 128 + ((lg ^ (lr & 7)) << 4), f1 = lr * 128 + (((lg + 4) ^ (lr & 7)) << 4);
    auto frag = [&](const uint8_t* base, int tile) {
        return join(*reinterpret_cast<const u32x4*>(base + tile * 2048 + f0), *reinterpret_cast<const u32x4*>(base + tile * 2048 + f1));
    };
    const auto as_float = [](int v) { return __builtin_bit_cast(float, v); };
    // One block of 128. On entry b holds its fragments of B and a the first one of A; every fragment is read from LDS one group
    // of matrix instructions before its use. With the last fragments of A in registers the stage is done with: the
    // waves meet (the next stage has arrived, NST - 2 younger ones are still on their way), the loads of stage k + NST start into
    // the buffer just freed, and the next step's first fragments are read under this step's last matrix instructions.
    constexpr int NL = NLA + NLB;
    int cur = 0;
    i32x8 b[TN], a;
    constexpr bool BOTH = SC == SCALE_F32_TILES;
    ScaleRange range;
    unsigned near = ~0u;
    auto step = [&](auto opc, int k) {
        constexpr int OP = decltype(opc)::value;
        const int buf = NST == 2 || NST == 4 ? OP % NST : cur, nbuf = NST == 2 || NST == 4 ? (OP + 1) % NST : cur + 1 == NST ? 0 : cur + 1;
        cur = nbuf;
        const uint8_t* la = lds[buf];
        const uint8_t* na = lds[nbuf];
        if constexpr (F32S) load_scales(min(k + 1, kb1 - 1), sa_next, sb_next);
        else if constexpr (OP == 1) load_scales(min(k + 3, kb1 - 1) >> 2, sa_next, sb_next);
        if constexpr (F32S) {
#pragma unroll
            for (int j = 0; j < TM; ++j) range.take((unsigned)sa[j]);
            if constexpr (BOTH) range.take((unsigned)sb[0]);
        } else if constexpr (!NATIVE && OP == 0) {
#pragma unroll
            for (int j = 0; j < TM; ++j) near &= bytes_near((unsigned)sa[j]);
#pragma unroll
            for (int i = 0; i < TN; ++i) near &= bytes_near((unsigned)sb[i]);
        }
        Wide bw[NATIVE ? 1 : TN];
        if constexpr (!NATIVE) {
#pragma unroll
            for (int i = 0; i < TN; ++i) bw[i] = widen<SM_FP8_E4M3>(b[i], F32S ? 1.f : byte_scale<OP>(sb[i]));
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            i32x8 next;
            if (j + 1 < TM) {
                next = frag(la, wm * TM + j + 1);
            } else {
                meet<(NST - 2) * NL>();
                stage(buf, min(k + NST, kb1 - 1));      // (behind the end: the last block again, read by nobody)
                next = frag(na, wm * TM);
            }
            f32x4 c[TN];
#pragma unroll
            for (int i = 0; i < TN; ++i) c[i] = F32S ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[i][j];
            if constexpr (!NATIVE) {
                mfma_wide<TN>(bw, widen<FA>(a, F32S ? 1.f : byte_scale<OP>(sa[j])), c);
            } else {
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    if constexpr (F32S) c[i] = mfma_block<0, FA>(b[i], a, c[i], 0x7f7f7f7f, 0x7f7f7f7f);
                    else c[i] = mfma_block<OP, FA>(b[i], a, c[i], sb[i], sa[j]);
                }
            }
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                if constexpr (F32S) {
                    // the block's sum on its own, then one multiply-add per element with sa[m] sb[n]
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float fa = as_float(sa[j]), fb = as_float(sb[SC == SCALE_F32_ROWS ? 4 * i + e : 0]);
                        acc[i][j][e] = BOTH ? fmaf(c[i][e], fa * fb, acc[i][j][e]) : fmaf(c[i][e] * fa, fb, acc[i][j][e]);
                    }
                } else {
                    acc[i][j] = c[i];
                }
                if (j + 1 == TM) b[i] = frag(na + BM * 128, wn * TN + i);
            }
            a = next;
        }
        if constexpr (F32S || OP == 3) take_scales();
    };
    if (kb0 < kb1) {
#pragma unroll
        for (int i = 0; i < NST; ++i) stage(i, min(kb0 + i, kb1 - 1));
        load_scales(F32S ? kb0 : kb0 >> 2, sa, sb);
        meet<(NST - 1) * NL>();
        a = frag(lds[0], wm * TM);
#pragma unroll
        for (int i = 0; i < TN; ++i) b[i] = frag(lds[0] + BM * 128, wn * TN + i);
        // kb0 is a multiple of 4: block kb's scale byte is byte kb % 4 of its dword, a constant of the unrolled step
        for (int kb = kb0; kb < kb1; kb += 4) {
            step(std::integral_constant<int, 0>{}, kb);
            if (kb + 1 < kb1) step(std::integral_constant<int, 1>{}, kb + 1);
            if (kb + 2 < kb1) step(std::integral_constant<int, 2>{}, kb + 2);
            if (kb + 3 < kb1) step(std::integral_constant<int, 3>{}, kb + 3);
        }
        meet<0>();      // no load into this block's LDS may outlive it
    }
    // Scales beyond the range are rare and known only once they are read: a wave that met one sums its share again, block by block
    // from memory, with the scales held apart. (A branch in every step keeps the matrix instructions from overlapping the
    // multiply-adds: 4096^3 123 -> 203 us.)
    if constexpr (F32S || !NATIVE) {
        if (__any(F32S ? range.far(BOTH) : (near & 0x80808080u) != 0x80808080u)) {
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            const auto codes = [&](const uint8_t* base, size_t pitch, int row, int kb) {
                const uint8_t* p = base + (size_t)row * pitch + (size_t)kb * 128 + lg * 16;
                return join(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + 64));
            };
            for (int kb = kb0; kb < kb1; ++kb) {
                load_scales(F32S ? kb : kb >> 2, sa, sb);
                const auto byte = [&](int dword) { return dword >> (8 * (kb & 3)) & 255; };
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    const i32x8 ca = codes(g.a, g.a_pitch, min(m0 + (wm * TM + j) * 16 + lr, g.M - 1), kb);
#pragma unroll
                    for (int i = 0; i < TN; ++i) {
                        const i32x8 cb = codes(g.b, g.b_pitch, min(n0 + (wn * TN + i) * 16 + lr, g.N - 1), kb);
                        f32x4 c = {0.f, 0.f, 0.f, 0.f};
                        if constexpr (NATIVE) {
                            c = mfma_block<0, FA>(cb, ca, c, 0x7f7f7f7f, 0x7f7f7f7f);
                        } else {
                            const Wide w = widen<SM_FP8_E4M3>(cb, 1.f);
                            mfma_wide<1>(&w, widen<FA>(ca, 1.f), &c);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (F32S) acc[i][j][e] += apart(c[e], as_float(sa[j]), as_float(sb[SC == SCALE_F32_ROWS ? 4 * i + e : 0]));
                            else acc[i][j][e] += apart(c[e], byte(sa[j]), byte(__shfl(sb[i], lg * 4 + e, 64)));      // (sb: of operand row lr)
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int m = m0 + (wm * TM + j) * 16 + lr;
        if (m >= g.M) continue;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int n = n0 + (wn * TN + i) * 16 + lg * 4;
            if (n >= g.N) continue;
            if (gridDim.y > 1) {
                float* o = g.ws + ((size_t)blockIdx.y * g.M + m) * g.N + n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < g.N) o[e] = acc[i][j][e];
            } else {
                store4(g, m, n, acc[i][j]);
            }
        }
    }
}

// (two waves per SIMD: left alone, the 128 x 128 tile with fp32 scales per row takes 300 registers and one)
template <int BM, int BN, int WM, int WN, int NST, int FA, int SC, bool NATIVE>
__global__ __launch_bounds__(WM* WN * 64, 2) void fp8_matmul_kernel(MatmulArgs g) {
    matmul_tile<BM, BN, WM, WN, NST, FA, SC, NATIVE>(g, blockIdx.x);
}

// Two products in one launch (a small layer's two gradients, neither of which fills the chip): the first blocks0 blocks are the
// first one's
template <int BM, int BN, int WM, int WN, int NST, int FA, int SC, bool NATIVE>
__global__ __launch_bounds__(WM* WN * 64) void fp8_matmul_pair_kernel(MatmulArgs g0, MatmulArgs g1, int blocks0) {
    const bool first = (int)blockIdx.x < blocks0;
    const MatmulArgs g = first ? g0 : g1;
    matmul_tile<BM, BN, WM, WN, NST, FA, SC, NATIVE>(g, first ? blockIdx.x : blockIdx.x - blocks0);
}

// Few rows of A (M <= 16 TM): the product is a stream through B, which is read once, straight into the matrix instructions'
// operand registers - no LDS, no barrier until the end. A block owns 16 TB rows of B; its eight waves take the blocks of 128
// along K in turn (together 1 KB of every row at a time) and U of them are in flight per wave. X: what A is - codes (SM_FP8_*
// + 8) or raw values (SM_TYPE_*), which every wave quantises on its way into the operand (their block maximum needs two
// cross-lane steps): one launch for a layer's forward pass. Bound by HBM: the codes of B; A comes from the caches once per
// block, which is why 16 and more rows of A take TB = 2 where B is long enough to fill the chip so.
constexpr int STREAM_WAVES = 8;
struct StreamArgs {
    MatmulArgs g;
    const void* x;          // raw rows (or null)
    size_t x_stride;
    int K;
};
// A lane's 32 raw values of block kb of row m -> codes and the block's scale byte (the same in the four lanes that share the
// row). r: the values as loaded; FULL = false: the row ends inside the block and they are read here.
template <int X, int RV, bool FULL>
__device__ __forceinline__ void quantize_rows(const StreamArgs& t, const u32x4* r, int kb, int m, int lg, i32x8& codes, int& byte) {
    float v[32];
    if constexpr (FULL) {
        unsigned top = 0;
#pragma unroll
        for (int q = 0; q < RV; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = mag_max<X>(top, mag<X>(r[q][i]));
        top = mag_both<X>(top);
        if (!__any(top >= inf_bits<X>)) {
            top = max(top, (unsigned)__shfl_xor((int)top, 16, 64));
            top = max(top, (unsigned)__shfl_xor((int)top, 32, 64));
            const int e = block_exponent(mag_float<X>(top), 8);
            byte = e + 127;
            if (!__any(e == -127)) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    unsigned d[8];
#pragma unroll
                    for (int i = 0; i < (RV == 8 ? 8 : 4); ++i) d[i] = RV == 8 ? r[2 * q + (i >> 2)][i & 3] : r[q][i];
                    const u32x2 w = codes8<X>(d, e, SM_FP8_E4M3, true);
                    codes[2 * q] = (int)w[0];
                    codes[2 * q + 1] = (int)w[1];
                }
                return;
            }
        }
#pragma unroll
        for (int q = 0; q < RV; ++q) unpack<X>(r[q], v + q * (32 / RV));
    } else {
        const int c = kb * 128 + lg * 16;
        const size_t row = (size_t)m * t.x_stride;
        load8<X>(t.x, row + c, t.K - c, v);
        load8<X>(t.x, row + c + 8, t.K - c - 8, v + 8);
        load8<X>(t.x, row + c + 64, t.K - c - 64, v + 16);
        load8<X>(t.x, row + c + 72, t.K - c - 72, v + 24);
    }
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) a = fmaxf(a, finite_abs(v[i]));
    a = fmaxf(a, __shfl_xor(a, 16, 64));
    a = fmaxf(a, __shfl_xor(a, 32, 64));
    const int e = block_exponent(a, 8);
    byte = e + 127;
    const float inv = inv_pow2(e);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const u32x2 w = cvt8(v + 8 * q, inv, SM_FP8_E4M3);
        codes[2 * q] = (int)w[0];
        codes[2 * q + 1] = (int)w[1];
    }
}

template <int X, int TM, int TB, bool F32S, bool NATIVE, int U>
__global__ __launch_bounds__(STREAM_WAVES * 64) void fp8_stream_kernel(StreamArgs t) {
    constexpr bool RAW = X < 8;
    constexpr int FA = X == 8 + SM_FP8_E5M2 ? SM_FP8_E5M2 : SM_FP8_E4M3;
    const MatmulArgs& g = t.g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lg = lane >> 4;
    const int n0 = blockIdx.x * 16 * TB;
    const int kb0 = blockIdx.y * g.kb_per_split, kb1 = min(g.KB, kb0 + g.kb_per_split);
    int brow[TB];
#pragma unroll
    for (int i = 0; i < TB; ++i) brow[i] = min(n0 + i * 16 + lr, g.N - 1);
    f32x4 acc[TM][TB];
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TB; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

    // NB blocks, STREAM_WAVES apart: all loads first, then the arithmetic. FULL: K covers the blocks (raw rows end inside the last one).
    constexpr int RV = RAW ? (X == SM_TYPE_F32 ? 8 : 4) : 2;       // 16-byte vectors of A per lane and block
    auto group = [&](auto nbc, auto fullc, int kb) {
        constexpr int NB = decltype(nbc)::value;
        constexpr bool FULL = decltype(fullc)::value;
        u32x4 bv[NB][TB][2], av[NB][TM][RV];
        int sb[NB][TB], sa[NB][TM];
        f32x4 fb[NB][TB];
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            const int k = kb + u * STREAM_WAVES;
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const uint8_t* bp = g.b + (size_t)brow[i] * g.b_pitch + (size_t)k * 128 + lg * 16;
                bv[u][i][0] = *reinterpret_cast<const u32x4*>(bp);
                bv[u][i][1] = *reinterpret_cast<const u32x4*>(bp + 64);
                if constexpr (F32S) {
                    const float* pb = static_cast<const float*>(g.bs) + (size_t)k * g.bs_rows;
#pragma unroll
                    for (int e = 0; e < 4; ++e) fb[u][i][e] = pb[min(n0 + i * 16 + lg * 4 + e, g.N - 1) >> g.b_shift];
                } else {
                    sb[u][i] = static_cast<const uint8_t*>(g.bs)[scale_at(k, brow[i] >> g.b_shift, g.bs_rows)];
                }
            }
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const int m = min(j * 16 + lr, g.M - 1);
                if constexpr (RAW) {
                    // the same places of the block as B's chunks: elements 16 lg ... + 15 and 64 + 16 lg ... + 15
                    const int c = k * 128 + lg * 16;
                    if constexpr (FULL) {
                        constexpr int ES = X == SM_TYPE_F32 ? 4 : 2;
                        const char* xp = static_cast<const char*>(t.x) + ((size_t)m * t.x_stride + c) * ES;
#pragma unroll
                        for (int q = 0; q < RV; ++q)
                            av[u][j][q] = *reinterpret_cast<const u32x4_u*>(xp + (q < RV / 2 ? q * 16 : 64 * ES + (q - RV / 2) * 16));
                    }
                } else {
                    const uint8_t* ap = g.a + (size_t)m * g.a_pitch + (size_t)k * 128 + lg * 16;
                    av[u][j][0] = *reinterpret_cast<const u32x4*>(ap);
                    av[u][j][1] = *reinterpret_cast<const u32x4*>(ap + 64);
                    if constexpr (F32S) sa[u][j] = __builtin_bit_cast(int, static_cast<const float*>(g.as)[(size_t)k * g.M + m]);
                    else sa[u][j] = static_cast<const uint8_t*>(g.as)[scale_at(k, m, g.M)];
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);      // (left alone the compiler sinks half of the loads between the products)
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            i32x8 bc[TB];
            Wide bw[NATIVE ? 1 : TB];
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                bc[i] = join(bv[u][i][0], bv[u][i][1]);
                if constexpr (!NATIVE) bw[i] = widen<SM_FP8_E4M3>(bc[i], F32S ? 1.f : __builtin_bit_cast(float, (unsigned)sb[u][i] << 23));
            }
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                i32x8 codes;
                int byte;
                if constexpr (RAW) {
                    quantize_rows<X, RV, FULL>(t, av[u][j], kb + u * STREAM_WAVES, min(j * 16 + lr, g.M - 1), lg, codes, byte);
                } else {
                    codes = join(av[u][j][0], av[u][j][1]);
                    byte = sa[u][j];
                }
                if constexpr (!F32S && !NATIVE) {
                    bool far = (unsigned)(byte - 32) >= 192;
#pragma unroll
                    for (int i = 0; i < TB; ++i) far |= (unsigned)(sb[u][i] - 32) >= 192;
                    if (__any(far)) {      // (bound by memory: the branch costs nothing here)
#pragma unroll
                        for (int i = 0; i < TB; ++i) {
                            const Wide w = widen<SM_FP8_E4M3>(bc[i], 1.f);
                            f32x4 c = {0.f, 0.f, 0.f, 0.f};
                            mfma_wide<1>(&w, widen<FA>(codes, 1.f), &c);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[j][i][e] += apart(c[e], byte, __shfl(sb[u][i], lg * 4 + e, 64));
                        }
                        continue;
                    }
                }
                f32x4 c[TB];
#pragma unroll
                for (int i = 0; i < TB; ++i) c[i] = F32S ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[j][i];
                if constexpr (NATIVE) {
#pragma unroll
                    for (int i = 0; i < TB; ++i) c[i] = mfma_block<0, FA>(bc[i], codes, c[i], sb[u][i], byte);
                } else {
                    mfma_wide<TB>(bw, widen<FA>(codes, F32S ? 1.f : __builtin_bit_cast(float, (unsigned)byte << 23)), c);
                }
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    if constexpr (F32S) {
                        const float fa = __builtin_bit_cast(float, byte);
                        ScaleRange range;
                        range.take((unsigned)byte);
                        if (__any(range.far(false))) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[j][i][e] += apart(c[i][e], fa, fb[u][i][e]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(c[i][e] * fa, fb[u][i][e], acc[j][i][e]);
                        }
                    } else {
                        acc[j][i] = c[i];
                    }
                }
            }
        }
    };
    constexpr std::integral_constant<bool, true> full{};
    const int kbf = RAW ? min(kb1, t.K >> 7) : kb1;       // blocks that K covers whole
    int kb = kb0 + wave;
    for (; kb + (U - 1) * STREAM_WAVES < kbf; kb += STREAM_WAVES * U) group(std::integral_constant<int, U>{}, full, kb);
    if constexpr (U > 2)
        for (; kb + STREAM_WAVES < kbf; kb += STREAM_WAVES * 2) group(std::integral_constant<int, 2>{}, full, kb);
    if constexpr (U > 1)
        for (; kb < kbf; kb += STREAM_WAVES) group(std::integral_constant<int, 1>{}, full, kb);
    if constexpr (RAW)
        if (kb < kb1) group(std::integral_constant<int, 1>{}, std::integral_constant<bool, false>{}, kb);
    // the waves' sums, added in their order
    __shared__ f32x4 part[STREAM_WAVES][TM * TB][64];
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TB; ++i) part[wave][j * TB + i][lane] = acc[j][i];
    __syncthreads();
    for (int q = wave; q < TM * TB; q += STREAM_WAVES) {
        f32x4 s = part[0][q][lane];
#pragma unroll
        for (int w = 1; w < STREAM_WAVES; ++w) s += part[w][q][lane];
        const int m = q / TB * 16 + lr, n = n0 + q % TB * 16 + lg * 4;
        if (m >= g.M || n >= g.N) continue;
        if (gridDim.y > 1) {
            float* o = g.ws + ((size_t)blockIdx.y * g.M + m) * g.N + n;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < g.N) o[e] = s[e];
        } else {
            store4(g, m, n, s);
        }
    }
}

// adds the slabs of a split product in their order and stores
__global__ __launch_bounds__(256) void fp8_matmul_reduce_kernel(MatmulArgs g, int splits) {
    const size_t per_row = (size_t)(g.N + 3) / 4;
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= per_row * g.M) return;
    const int m = (int)(id / per_row), n = (int)(id % per_row) * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < splits; ++k) {
        const float* p = g.ws + ((size_t)k * g.M + m) * g.N + n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < g.N) s[e] += p[e];
    }
    store4(g, m, n, s);
}

// nothing to sum: zeros (or out as it is, when adding to it)
__global__ __launch_bounds__(256) void fp8_matmul_empty_kernel(MatmulArgs g) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t per_row = (size_t)(g.N + 3) / 4;
    if (id < per_row * g.M) store4(g, (int)(id / per_row), (int)(id % per_row) * 4, f32x4{0.f, 0.f, 0.f, 0.f});
}

// Which kernel takes an M x N x 128 KB product, and in how many slices of K. Measured on MI355X (us):
//                                        256 x 256   256 x 128   128 x 128   64 x 64
//   8192^3      fast sums, 2^e scales          413         488         499       921
//   4096^3      fast sums, 2^e scales           59          71          70       126
//   4096^3      f16 result, fp32 scales        317         124         133       201   (256 x 256 spills)
//   2048^3      fast sums, 2^e scales           33          22          17        18
//   512 x 4096 x 4096, fast sums                50          31          26        18
// A 256-row tile takes a CU, two 128 x 128 tiles share one: the large tile is taken where its rounds over the 256 CUs are not
// emptier than the small one's by more than what it gains (1.2 x); below 192 tiles of 128 x 128 the chip is filled with
// 64 x 64 ones, and where even those are few (a weight gradient of small layers) K is split, at least eight blocks a slice, and
// the slices are added by a second kernel (128 x 256 x 8192: 27 us in one slice).
// Up to 32 rows the stream kernel, which needs no LDS and keeps more of B in flight (32 x 4096 x 4096, fast sums: 9.6 against 12.3 us);
// above, its rereads of A through the caches cost more (37 x 8200 x 5001, fast sums: 25 against 20 us).
enum { TILE_STREAM, TILE_64, TILE_128, TILE_256 };
struct Plan {
    int kind, splits, kb_per_split;
    bool fast;      // SM_FP8_FAST_SUM
};
static Plan matmul_plan(int M, int N, int KB) {
    const auto tiles = [&](long long bm, long long bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
    const auto fill = [](long long t, long long slots) { return (double)t / (double)((t + slots - 1) / slots * slots); };
    Plan p{TILE_64, 1, KB, false};
    long long t = tiles(64, 64);
    if (M <= 32) {
        p.kind = TILE_STREAM;
        t = (N + 15) / 16;
    } else if (tiles(128, 128) >= 192) {
        p.kind = 1.2 * fill(tiles(256, 256), 256) >= fill(tiles(128, 128), 512) ? TILE_256 : TILE_128;
        return p;
    }
    if (t <= (p.kind == TILE_STREAM ? 128 : 192) && KB >= 16) {
        const long long want = std::min<long long>(384 / t, KB / (p.kind == TILE_STREAM ? 32 : 8));
        if (want > 1) {
            p.kb_per_split = (int)((KB + want - 1) / want + 3) / 4 * 4;      // (whole dwords of scale bytes)
            p.splits = (KB + p.kb_per_split - 1) / p.kb_per_split;
        }
    }
    return p;
}

// A result's type, and whether its sums may run on the 8-bit matrix instruction. That instruction (both its forms) aligns the
// products of eight neighbouring k to the largest of them and keeps 13 bits below its leading one (measured, not documented), fp32
// beyond that: each of the other seven loses up to 2^-13 of the largest, so a sum is off by up to 7 * 2^-13 of sum |a||b|
// beside what fp32 loses - of the terms' magnitudes, not of the result, which may be far smaller (rms at K = 128: 2^-19 of it for
// normal data, 2^-15 for log-normal of sigma 2, falling with sqrt(K)). Those are fewer bits than a sum is owed, so it is taken
// where the caller asks for it only, and only for bf16 results. Every other product widens the codes to bf16 and sums in
// fp32: us, fast against that, 8192^3 463 / 876, layer backward 4096^3 208 / 260, 37 x 5001 -> 8200 21.0 / 22.4, 1 x 4096 -> 4096 6.1 / 6.7.
struct ResultType {
    int type;
    bool fast, ok;
};
static ResultType result_type(int t) {
    const int type = t & ~SM_FP8_FAST_SUM;
    const bool fast = t != type;
    return {type, fast, type >= 0 && type <= SM_TYPE_F16 && (!fast || type == SM_TYPE_BF16)};
}

template <int X, int TM, int TB, bool F32S, bool NATIVE, int U>
static void launch_stream(const StreamArgs& t, int splits, hipStream_t s) {
    hipLaunchKernelGGL((fp8_stream_kernel<X, TM, TB, F32S, NATIVE, U>), dim3((unsigned)((t.g.N + 16 * TB - 1) / (16 * TB)), (unsigned)splits),
                       dim3(STREAM_WAVES * 64), 0, s, t);
}
template <int X>
static void launch_stream_raw(const StreamArgs& t, bool fast, int splits, hipStream_t s) {
    constexpr int U = X == SM_TYPE_F32 ? 2 : 4;
    if (fast) launch_stream<X, 1, 1, false, true, U>(t, splits, s);
    else launch_stream<X, 1, 1, false, false, U>(t, splits, s);
}
template <int X, bool NATIVE>
static void launch_stream_pow2(const StreamArgs& t, int splits, hipStream_t s) {
    const bool wide = (t.g.N + 31) / 32 >= 192;       // 32 rows of B per block still fill the chip
    if (t.g.M <= 16) launch_stream<X, 1, 1, false, NATIVE, 4>(t, splits, s);
    else wide ? launch_stream<X, 2, 2, false, NATIVE, 2>(t, splits, s) : launch_stream<X, 2, 1, false, NATIVE, 2>(t, splits, s);
}
template <int X>
static void launch_stream_codes(const StreamArgs& t, bool f32s, bool fast, int splits, hipStream_t s) {
    if (!f32s) {
        if (fast) launch_stream_pow2<X, true>(t, splits, s);
        else launch_stream_pow2<X, false>(t, splits, s);
    } else if (t.g.M <= 16) launch_stream<X, 1, 1, true, false, 4>(t, splits, s);
    else launch_stream<X, 2, 1, true, false, 2>(t, splits, s);
}
static void launch_reduce(const MatmulArgs& g, int splits, hipStream_t s) {
    const size_t quads = (size_t)(g.N + 3) / 4 * g.M;
    hipLaunchKernelGGL(fp8_matmul_reduce_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, g, splits);
}

template <int BM, int BN, int WM, int WN, int NST, bool NATIVE, bool F32S>
static void launch_matmul(const MatmulArgs& g, int a_fmt, int splits, hipStream_t s) {
    const dim3 grid((unsigned)(((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN)), (unsigned)splits), block(WM * WN * 64);
    const auto go = [&](auto fa, auto sc) {
        hipLaunchKernelGGL((fp8_matmul_kernel<BM, BN, WM, WN, NST, decltype(fa)::value, decltype(sc)::value, NATIVE>), grid, block, 0, s, g);
    };
    const auto with_format = [&](auto sc) {
        if (a_fmt == SM_FP8_E4M3) go(std::integral_constant<int, SM_FP8_E4M3>{}, sc);
        else go(std::integral_constant<int, SM_FP8_E5M2>{}, sc);
    };
    if constexpr (!F32S) with_format(std::integral_constant<int, SCALE_POW2>{});
    else if (g.b_shift == 0) with_format(std::integral_constant<int, SCALE_F32_ROWS>{});
    else with_format(std::integral_constant<int, SCALE_F32_TILES>{});
}

template <bool NATIVE>
static void launch_tile(int kind, const MatmulArgs& g, int a_fmt, bool f32s, int splits, hipStream_t s) {
    // Widened codes with power-of-two scales stay with the smaller tile: two blocks a CU convert and multiply in turn, and 256 x 256
    // spills (us, 128 x 128 against 256 x 256, fp32 result: 8192 x 8192 x 1024 176 / 206, x 2048 284 / 306, x 4096 534 / 528;
    // 4096 x 11008 x 4096 343 / 353; 4096 x 4096 x 4096 123 / 121, x 8192 230 / 220).
    if (kind == TILE_256 && f32s) return launch_matmul<256, 128, 4, 2, 2, NATIVE, true>(g, a_fmt, splits, s);
    if constexpr (NATIVE)
        if (kind == TILE_256) return launch_matmul<256, 256, 2, 4, 2, NATIVE, false>(g, a_fmt, splits, s);
    // A ring of four stages lets two blocks share a CU, one of three stages three: taken where two a CU would leave a second round
    // (1500 x 1500 x 700 fp32 12.6 -> 10.8 us, 1600 x 1600 x 2000 21.4 -> 18.8; below 512 tiles +-2 %, 128 x 8192 x 4096 12.4 -> 13.6).
    const bool three = (long long)((g.M + 63) / 64) * ((g.N + 63) / 64) * splits > 512;
    if (kind != TILE_64 && !f32s) launch_matmul<128, 128, 2, 2, 2, NATIVE, false>(g, a_fmt, splits, s);
    else if (kind != TILE_64) launch_matmul<128, 128, 2, 2, 2, NATIVE, true>(g, a_fmt, splits, s);
    else if (!three && !f32s) launch_matmul<64, 64, 2, 2, 4, NATIVE, false>(g, a_fmt, splits, s);
    else if (!three) launch_matmul<64, 64, 2, 2, 4, NATIVE, true>(g, a_fmt, splits, s);
    else if (!f32s) launch_matmul<64, 64, 2, 2, 3, NATIVE, false>(g, a_fmt, splits, s);
    else launch_matmul<64, 64, 2, 2, 3, NATIVE, true>(g, a_fmt, splits, s);
}

template <int T>
static int launch_quantize(const QuantArgs& a, int tiles, hipStream_t s) {
    const unsigned cb = (unsigned)((a.cols + 127) / 128);
    const dim3 grid(cb, (unsigned)((a.rows + 127) / 128));
    const bool q = a.q != nullptr, qt = a.qt != nullptr;
    if (tiles) {
        if (q && qt) hipLaunchKernelGGL((fp8_quantize_kernel<T, true, true, true, 4, 128>), grid, dim3(512), 0, s, a);
        else if (q) hipLaunchKernelGGL((fp8_quantize_kernel<T, true, true, false, 4, 128>), grid, dim3(512), 0, s, a);
        else hipLaunchKernelGGL((fp8_quantize_kernel<T, true, false, true, 4, 128>), grid, dim3(512), 0, s, a);
    } else {
        const size_t n = (size_t)grid.x * grid.y;
        // fewer tiles of 128 x 128 than half the CUs: small blocks (fp32 / bf16, both ways, us: 300 x 300 6.1 -> 4.6 / 6.2 -> 4.1,
        // 1029 x 517 6.5 -> 5.5 / 7.4 -> 5.2, 1024 x 1024 6.5 -> 5.8 / 6.0 -> 4.8; 2048 x 1536 9.1 -> 10.1 / 7.2 -> 8.3)
        if (qt && n < 128) {
            const unsigned bq = q ? cb * (unsigned)((a.rows + 15) / 16) : 0;
            const unsigned bt = (unsigned)((a.cols + 31) / 32) * grid.y;
            hipLaunchKernelGGL(fp8_quantize_small_kernel<T>, dim3(bq + bt), dim3(256), 0, s, a, (int)bq);
        } else if (q && qt) hipLaunchKernelGGL((fp8_quantize_kernel<T, false, true, true, 4, 128>), grid, dim3(512), 0, s, a);
        else if (qt) hipLaunchKernelGGL((fp8_quantize_kernel<T, false, false, true, 4, 128>), grid, dim3(512), 0, s, a);
        else if (n >= 1024) hipLaunchKernelGGL((fp8_quantize_kernel<T, false, true, false, 8, 128>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((fp8_quantize_kernel<T, false, true, false, 1, 16>), dim3(cb, (unsigned)((a.rows + 15) / 16)), dim3(256), 0, s, a);
    }
    SM_LAUNCH_CHECK();
    return 0;
}

}  // namespace sm

extern "C" {

static constexpr int MAX_QUANTIZED = 65535 * 128;      // rows / columns of a quantised matrix: the grid's second dimension, in 128s

int sm_fp8_quantize(const void* x, int x_type, int rows, int cols, size_t x_stride, int fmt, int tiles, void* q, void* q_scale,
                    void* qt, void* qt_scale, void* stream) {
    if (rows < 0 || cols < 0 || x_type < 0 || x_type > SM_TYPE_F16 || (fmt != SM_FP8_E4M3 && fmt != SM_FP8_E5M2) ||
        (q == nullptr) != (q_scale == nullptr) || (qt == nullptr) != (qt_scale == nullptr) || (q == nullptr && qt == nullptr))
        return (int)hipErrorInvalidValue;
    if (rows == 0 || cols == 0) return 0;
    if (x == nullptr || x_stride < (size_t)cols || rows > MAX_QUANTIZED || cols > MAX_QUANTIZED || (uintptr_t)q % 16 || (uintptr_t)qt % 16)
        return (int)hipErrorInvalidValue;
    const sm::QuantArgs a{x, x_stride, rows, cols, fmt, (uint8_t*)q, (uint8_t*)q_scale, (uint8_t*)qt, (uint8_t*)qt_scale};
    hipStream_t s = (hipStream_t)stream;
    if (x_type == SM_TYPE_F32) return sm::launch_quantize<SM_TYPE_F32>(a, tiles, s);
    if (x_type == SM_TYPE_BF16) return sm::launch_quantize<SM_TYPE_BF16>(a, tiles, s);
    return sm::launch_quantize<SM_TYPE_F16>(a, tiles, s);
}

size_t sm_fp8_matmul_ws_bytes(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const sm::Plan p = sm::matmul_plan(M, N, (int)(((size_t)K + 127) / 128));
    return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) : 0;
}

// offsets from a tile's first row (256 rows) and from a row of scales are 32 bits
static constexpr size_t MAX_PITCH = 0xfffff0;
static constexpr int MAX_ROWS = (1 << 30) - 1;

// checks a product's arguments and plans it (M, N, K > 0)
static int prepare_product(sm::MatmulArgs& g, sm::Plan& p, const void* a, const void* a_scale, int a_fmt, size_t a_pitch, const void* b,
                           const void* b_scale, int b_tiles, size_t b_pitch, int M, int N, int K, void* out, int out_type, size_t out_stride,
                           int accumulate, void* ws, size_t ws_bytes) {
    const int KB = (int)(((size_t)K + 127) / 128);
    const sm::ResultType rt = sm::result_type(out_type);
    if (!rt.ok || (a_fmt != SM_FP8_E4M3 && a_fmt != SM_FP8_E5M2) || out == nullptr || out_stride < (size_t)N ||
        a == nullptr || b == nullptr || a_scale == nullptr || b_scale == nullptr || a_pitch < (size_t)KB * 128 || b_pitch < (size_t)KB * 128 ||
        a_pitch % 16 || b_pitch % 16 || (uintptr_t)a % 16 || (uintptr_t)b % 16 || (uintptr_t)a_scale % 4 || (uintptr_t)b_scale % 4 ||
        a_pitch > MAX_PITCH || b_pitch > MAX_PITCH || M > MAX_ROWS || N > MAX_ROWS)
        return (int)hipErrorInvalidValue;
    p = sm::matmul_plan(M, N, KB);
    p.fast = rt.fast;
    if (p.splits > 1 && (ws == nullptr || ws_bytes < (size_t)p.splits * M * N * sizeof(float))) return (int)hipErrorInvalidValue;
    g = sm::MatmulArgs{(const uint8_t*)a, (const uint8_t*)b, a_scale, b_scale, out, (float*)ws, a_pitch, b_pitch, out_stride, M, N, KB,
                       b_tiles ? 7 : 0, b_tiles ? (N + 127) / 128 : N, rt.type, accumulate, p.kb_per_split};
    return 0;
}

static int run_product(const sm::MatmulArgs& g, const sm::Plan& p, int a_fmt, bool f32s, int K, hipStream_t s) {
    if (p.kind == sm::TILE_STREAM) {
        const sm::StreamArgs t{g, nullptr, 0, K};
        if (a_fmt == SM_FP8_E4M3) sm::launch_stream_codes<8 + SM_FP8_E4M3>(t, f32s, p.fast, p.splits, s);
        else sm::launch_stream_codes<8 + SM_FP8_E5M2>(t, f32s, p.fast, p.splits, s);
    } else if (p.fast) {
        sm::launch_tile<true>(p.kind, g, a_fmt, f32s, p.splits, s);
    } else {
        sm::launch_tile<false>(p.kind, g, a_fmt, f32s, p.splits, s);
    }
    SM_LAUNCH_CHECK();
    if (p.splits > 1) sm::launch_reduce(g, p.splits, s);
    SM_LAUNCH_CHECK();
    return 0;
}

int sm_fp8_matmul(const void* a, const void* a_scale, int a_fmt, size_t a_pitch, const void* b, const void* b_scale, int b_tiles,
                  size_t b_pitch, int scale_f32, int M, int N, int K, void* out, int out_type, size_t out_stride, int accumulate,
                  void* ws, size_t ws_bytes, void* stream) {
    const sm::ResultType rt = sm::result_type(out_type);
    if (M < 0 || N < 0 || K < 0 || !rt.ok || (a_fmt != SM_FP8_E4M3 && a_fmt != SM_FP8_E5M2)) return (int)hipErrorInvalidValue;
    if (M == 0 || N == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    sm::MatmulArgs g{};
    if (K == 0) {
        if (out == nullptr || out_stride < (size_t)N) return (int)hipErrorInvalidValue;
        g.out = out;
        g.out_stride = out_stride;
        g.M = M;
        g.N = N;
        g.out_type = rt.type;
        const size_t quads = (size_t)(N + 3) / 4 * M;
        if (!accumulate) hipLaunchKernelGGL(sm::fp8_matmul_empty_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, g);
        SM_LAUNCH_CHECK();
        return 0;
    }
    sm::Plan p;
    if (const int e = prepare_product(g, p, a, a_scale, a_fmt, a_pitch, b, b_scale, b_tiles, b_pitch, M, N, K, out, out_type, out_stride, accumulate,
                                      ws, ws_bytes))
        return e;
    return run_product(g, p, a_fmt, scale_f32 != 0, K, s);
}

// rows up to which a layer's forward pass quantises inside the product
static constexpr int LINEAR_FUSED_ROWS = 16;

size_t sm_fp8_linear_ws_bytes(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const size_t slabs = sm_fp8_matmul_ws_bytes(M, N, K);
    if (M <= LINEAR_FUSED_ROWS) return slabs;
    const size_t KB = ((size_t)K + 127) / 128;
    return (slabs + 15) / 16 * 16 + (size_t)M * KB * 128 + (KB + 3) / 4 * M * 4;
}

int sm_fp8_linear(const void* x, int x_type, size_t x_stride, const void* w, const void* w_scale, int w_tiles, size_t w_pitch, int M,
                  int N, int K, void* out, int out_type, size_t out_stride, void* ws, size_t ws_bytes, void* stream) {
    const sm::ResultType rt = sm::result_type(out_type);
    if (M < 0 || N < 0 || K < 0 || x_type < 0 || x_type > SM_TYPE_F16 || !rt.ok) return (int)hipErrorInvalidValue;
    if (M == 0 || N == 0) return 0;
    if (K > 0 && (x == nullptr || x_stride < (size_t)K || (ws == nullptr && sm_fp8_linear_ws_bytes(M, N, K) > 0) ||
                  ws_bytes < sm_fp8_linear_ws_bytes(M, N, K) || (uintptr_t)ws % 16))
        return (int)hipErrorInvalidValue;
    const int KB = (int)(((size_t)K + 127) / 128);
    if (K == 0 || M > LINEAR_FUSED_ROWS) {
        const size_t slabs = (sm_fp8_matmul_ws_bytes(M, N, K) + 15) / 16 * 16;
        char* q = (char*)ws + slabs;
        char* qs = q + (size_t)M * KB * 128;
        if (K > 0)
            if (const int e = sm_fp8_quantize(x, x_type, M, K, x_stride, SM_FP8_E4M3, 0, q, qs, nullptr, nullptr, stream)) return e;
        return sm_fp8_matmul(q, qs, SM_FP8_E4M3, (size_t)KB * 128, w, w_scale, w_tiles, w_pitch, 0, M, N, K, out, out_type, out_stride, 0,
                             ws, slabs, stream);
    }
    if (out == nullptr || out_stride < (size_t)N || w == nullptr || w_scale == nullptr || w_pitch < (size_t)KB * 128 || w_pitch % 16 ||
        (uintptr_t)w % 16 || N > MAX_ROWS)
        return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    const sm::Plan p = sm::matmul_plan(M, N, KB);
    sm::StreamArgs t{{nullptr, (const uint8_t*)w, nullptr, w_scale, out, (float*)ws, 0, w_pitch, out_stride, M, N, KB, w_tiles ? 7 : 0,
                      w_tiles ? (N + 127) / 128 : N, rt.type, 0, p.kb_per_split}, x, x_stride, K};
    if (x_type == SM_TYPE_F32) sm::launch_stream_raw<SM_TYPE_F32>(t, rt.fast, p.splits, s);
    else if (x_type == SM_TYPE_BF16) sm::launch_stream_raw<SM_TYPE_BF16>(t, rt.fast, p.splits, s);
    else sm::launch_stream_raw<SM_TYPE_F16>(t, rt.fast, p.splits, s);
    SM_LAUNCH_CHECK();
    if (p.splits > 1) sm::launch_reduce(t.g, p.splits, s);
    SM_LAUNCH_CHECK();
    return 0;
}

// workspace of a backward pass: both quantised forms of dy, then one product's slabs (the products run one after the other)
static size_t bwd_layout(int M, int N, int K, bool need_dx, bool need_dw, size_t* qs, size_t* t, size_t* ts, size_t* slabs) {
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t nb = ((size_t)N + 127) / 128, mb = ((size_t)M + 127) / 128;
    size_t at = 0;
    if (need_dx) {
        at = up((size_t)M * nb * 128);
        *qs = at;
        at += up((nb + 3) / 4 * M * 4);
    }
    *t = at;
    if (need_dw) {
        at += up((size_t)N * mb * 128);
        *ts = at;
        at += up((mb + 3) / 4 * N * 4);
    }
    *slabs = at;
    return at + std::max(need_dx ? sm_fp8_matmul_ws_bytes(M, K, N) : 0, need_dw ? sm_fp8_matmul_ws_bytes(N, K, M) : 0);
}

size_t sm_fp8_linear_backward_ws_bytes(int M, int N, int K, int need_dx, int need_dw) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    size_t qs, t, ts, slabs;
    return bwd_layout(M, N, K, need_dx != 0, need_dw != 0, &qs, &t, &ts, &slabs);
}

int sm_fp8_linear_backward(const void* dy, int dy_type, size_t dy_stride, int fmt, int M, int N, int K, const void* wt, const void* wt_scale,
                           int wt_tiles, size_t wt_pitch, const void* xt, const void* xt_scale, int xt_tiles, size_t xt_pitch, void* dx,
                           int dx_type, size_t dx_stride, float* dw, size_t dw_stride, int accumulate, void* ws, size_t ws_bytes, void* stream) {
    if (M <= 0 || N <= 0 || K <= 0 || (dx == nullptr && dw == nullptr)) return (int)hipErrorInvalidValue;
    size_t qs = 0, t = 0, ts = 0, slabs = 0;
    if (ws == nullptr || (uintptr_t)ws % 16 || ws_bytes < bwd_layout(M, N, K, dx != nullptr, dw != nullptr, &qs, &t, &ts, &slabs))
        return (int)hipErrorInvalidValue;
    char* w = (char*)ws;
    const hipStream_t s = (hipStream_t)stream;
    sm::MatmulArgs gx{}, gw{};
    sm::Plan px{}, pw{};
    if (dx)
        if (const int e = prepare_product(gx, px, w, w + qs, fmt, ((size_t)N + 127) / 128 * 128, wt, wt_scale, wt_tiles, wt_pitch, M, K, N, dx, dx_type,
                                          dx_stride, 0, w + slabs, ws_bytes - slabs))
            return e;
    if (dw)
        if (const int e = prepare_product(gw, pw, w + t, w + ts, fmt, ((size_t)M + 127) / 128 * 128, xt, xt_scale, xt_tiles, xt_pitch, N, K, M, dw,
                                          SM_TYPE_F32, dw_stride, accumulate, w + slabs, ws_bytes - slabs))
            return e;
    if (const int e = sm_fp8_quantize(dy, dy_type, M, N, dy_stride, fmt, 0, dx ? w : nullptr, dx ? w + qs : nullptr, dw ? w + t : nullptr,
                                      dw ? w + ts : nullptr, stream))
        return e;
    // two products of small tiles, neither of which fills the chip: one launch (1029 x 517 x 1283: 8.3 + 8.2 -> 10.7 us, of which a
    // ring of three stages - three blocks a CU instead of two - is worth 1.1 and the order below 1)
    if (dx && dw && px.kind == sm::TILE_64 && pw.kind == sm::TILE_64 && px.splits == 1 && pw.splits == 1 && !px.fast) {
        // the one with more blocks of K first: its tiles run longest, and the last tiles to start should be short
        const bool swap = gw.KB > gx.KB;
        const sm::MatmulArgs &g0 = swap ? gw : gx, &g1 = swap ? gx : gw;
        const int b0 = ((g0.M + 63) / 64) * ((g0.N + 63) / 64), b1 = ((g1.M + 63) / 64) * ((g1.N + 63) / 64);
        if (fmt == SM_FP8_E4M3)
            hipLaunchKernelGGL((sm::fp8_matmul_pair_kernel<64, 64, 2, 2, 3, SM_FP8_E4M3, sm::SCALE_POW2, false>), dim3((unsigned)(b0 + b1)), dim3(256),
                               0, s, g0, g1, b0);
        else
            hipLaunchKernelGGL((sm::fp8_matmul_pair_kernel<64, 64, 2, 2, 3, SM_FP8_E5M2, sm::SCALE_POW2, false>), dim3((unsigned)(b0 + b1)), dim3(256),
                               0, s, g0, g1, b0);
        SM_LAUNCH_CHECK();
        return 0;
    }
    if (dx)
        if (const int e = run_product(gx, px, fmt, false, N, s)) return e;
    if (dw) return run_product(gw, pw, fmt, false, M, s);
    return 0;
}

}  // extern "C"
