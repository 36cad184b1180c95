// F8: 8-bit floating point with one scale per block of 128 - the quantiser and the matrix product (include/stylemesh_hip.h
// section F8). The reference computes in fp32 throughout and has no counterpart; the format is the next rung below this
// library's fp16x2 arithmetic (conv_split_kernel.h) and keeps its idea: operands scaled by powers of two.
//
//   x[r][c] = code[r][c] * 2^(s - 127)   codes e4m3 (largest 448) or e5m2 (57344), s = one byte per 128 columns of a row
//                                        ("rows") or per 128 x 128 tile ("tiles")
//   product: out[m][n] = sum_kb sa[m][kb] sb[n or n / 128][kb] sum_{k in block kb} a[m][k] b[n][k], fp32 accumulate
//
// Power-of-two scales make the quantiser exact up to the one rounding to 8 bits (x 2^-e is exact) and let the matrix
// cores apply the scales themselves: v_mfma_scale_f32_16x16x128_f8f6f4 takes a block of 128 per instruction and one scale
// byte per operand row, so a scaled block costs no vector instruction. fp32 scales (any value) take the same kernels with
// the block's partial sum multiplied in on the vector unit.
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

// eight consecutive elements of a row as fp32 (type: SM_TYPE_*); `valid` of them exist, the others are 0
template <int T>
__device__ __forceinline__ void load8(const void* base, size_t off, int valid, float* v) {
    if (valid >= 8) {
        if constexpr (T == SM_TYPE_F32) {
            const u32x4_u* p = reinterpret_cast<const u32x4_u*>(static_cast<const float*>(base) + off);
            const u32x4 a = p[0], b = p[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = __builtin_bit_cast(float, (unsigned)a[j]);
                v[4 + j] = __builtin_bit_cast(float, (unsigned)b[j]);
            }
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4_u*>(static_cast<const uint16_t*>(base) + off);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned lo = a[j] & 0xffffu, hi = a[j] >> 16;
                v[2 * j] = T == SM_TYPE_BF16 ? bf16_to_f32(lo) : f16_to_f32(lo);
                v[2 * j + 1] = T == SM_TYPE_BF16 ? bf16_to_f32(hi) : f16_to_f32(hi);
            }
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

// One 128 x 128 tile per block of 256 threads: thread t holds rows 8 (t / 16) ... + 7, columns 8 (t % 16) ... + 7 in registers
// (x is read once whatever is produced). Row maxima: 16 lanes of a row; column maxima: registers, then the wave's four row
// groups, then the four waves through LDS; tile maximum: all. The transposed codes go through a 128 x (128 + 16) byte LDS
// image so that both results leave as whole 128-byte lines.
// Bound by HBM: cols * rows * (sizeof(x) + 1 per result).
template <int T, bool TILES, bool Q, bool QT>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(QuantArgs a) {
    const int tid = threadIdx.x, rg = tid >> 4, cg = tid & 15, wave = tid >> 6;
    const int tr = blockIdx.y * 128, tc = blockIdx.x * 128;
    const int top = a.fmt == SM_FP8_E4M3 ? 8 : 15;
    const int c0 = tc + cg * 8;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = tr + rg * 8 + i;
        load8<T>(a.x, (size_t)r * a.stride + c0, r < a.rows ? a.cols - c0 : 0, v[i]);
    }
    __shared__ float red[4][128];
    __shared__ __align__(16) uint8_t img[QT ? 128 * 144 : 16];
    float rmax[8], cmax[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[i][j]));
        if (!TILES && Q) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        }
        rmax[i] = m;
    }
    const int cblocks = (a.cols + 127) >> 7, rblocks = (a.rows + 127) >> 7;
    int tile_e = 0;
    if constexpr (TILES) {
        float m = rmax[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, rmax[i]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        if ((tid & 63) == 0) red[wave][0] = m;
        __syncthreads();
        tile_e = block_exponent(fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])), top);
        if (tid < 4) {      // thread 0: this tile's byte; the row's / column's last tile also fills the dword's unused bytes
            if (Q && (tid == 0 || ((int)blockIdx.x + tid < (cblocks + 3) / 4 * 4 && (int)blockIdx.x == cblocks - 1)))
                a.qs[scale_at(blockIdx.x + tid, blockIdx.y, rblocks)] = tid == 0 ? (uint8_t)(tile_e + 127) : (uint8_t)127;
            if (QT && (tid == 0 || ((int)blockIdx.y + tid < (rblocks + 3) / 4 * 4 && (int)blockIdx.y == rblocks - 1)))
                a.qts[scale_at(blockIdx.y + tid, blockIdx.x, cblocks)] = tid == 0 ? (uint8_t)(tile_e + 127) : (uint8_t)127;
        }
    }
    if constexpr (Q) {
        const size_t pitch = (size_t)cblocks * 128;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = tr + rg * 8 + i;
            const int e = TILES ? tile_e : block_exponent(rmax[i], top);
            if (r < a.rows) {
                *reinterpret_cast<u32x2*>(a.q + (size_t)r * pitch + c0) = cvt8(v[i], inv_pow2(e), a.fmt);
                if (!TILES && cg < 4 && (cg == 0 || ((int)blockIdx.x == cblocks - 1 && (int)blockIdx.x + cg < (cblocks + 3) / 4 * 4)))
                    a.qs[scale_at(blockIdx.x + cg, r, a.rows)] = cg == 0 ? (uint8_t)(e + 127) : (uint8_t)127;
            }
        }
    }
    if constexpr (QT) {
        if constexpr (!TILES) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[i][j]));
                m = fmaxf(m, __shfl_xor(m, 16, 64));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                cmax[j] = m;
            }
            if ((tid & 63) < 16) {
#pragma unroll
                for (int j = 0; j < 8; ++j) red[wave][cg * 8 + j] = cmax[j];
            }
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int cl = cg * 8 + j;
            int e = tile_e;
            if (!TILES) {
                e = block_exponent(fmaxf(fmaxf(red[0][cl], red[1][cl]), fmaxf(red[2][cl], red[3][cl])), top);
                if (tc + cl < a.cols && rg < 4 && (rg == 0 || ((int)blockIdx.y == rblocks - 1 && (int)blockIdx.y + rg < (rblocks + 3) / 4 * 4)))
                    a.qts[scale_at(blockIdx.y + rg, tc + cl, a.cols)] = rg == 0 ? (uint8_t)(e + 127) : (uint8_t)127;
            }
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = v[i][j];
            *reinterpret_cast<u32x2*>(img + cl * 144 + rg * 8) = cvt8(t, inv_pow2(e), a.fmt);
        }
        __syncthreads();
        const size_t pitch = (size_t)rblocks * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {      // 8 lanes write a column's 128 bytes
            const int cl = i * 32 + (tid >> 3);
            if (tc + cl < a.cols)
                *reinterpret_cast<u32x4*>(a.qt + (size_t)(tc + cl) * pitch + tr + (tid & 7) * 16) =
                    *reinterpret_cast<const u32x4*>(img + cl * 144 + (tid & 7) * 16);
        }
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

__device__ __forceinline__ void store4(const MatmulArgs& g, int m, int n, f32x4 v) {
    const int cnt = g.N - n;
    if (g.out_type == SM_TYPE_F32) {
        float* o = static_cast<float*>(g.out) + (size_t)m * g.out_stride + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cnt) o[j] = g.accumulate ? o[j] + v[j] : v[j];
    } else {
        uint16_t* o = static_cast<uint16_t*>(g.out) + (size_t)m * g.out_stride + n;
        const bool bf = g.out_type == SM_TYPE_BF16;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cnt) {
                float x = v[j];
                if (g.accumulate) x += bf ? bf16_to_f32(o[j]) : f16_to_f32(o[j]);
                o[j] = (uint16_t)(bf ? f32_to_bf16(x) : f32_to_f16(x));
            }
    }
}

// direct loads into LDS are counted as vector-memory operations: a wave waits for its own before the barrier that hands
// the stage to the others
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// An operand's 32 codes of a lane as bf16, scaled by 2^(byte - 127): e4m3 / e5m2 have 4 / 3 significant bits, bf16 has 8 and
// fp32's exponents, so this is exact. scale: the byte in the exponent field of a float.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
struct Wide {
    bf16x8 p[4];
};
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
__device__ __forceinline__ f32x4 mfma_wide(const Wide& b, const Wide& a, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[i], a.p[i], c, 0, 0, 0);
    return c;
}

template <int OP, int FA>
__device__ __forceinline__ f32x4 mfma_block(i32x8 bfrag, i32x8 afrag, f32x4 c, int sb, int sa) {
    // first operand = rows of b (the result's rows), second = rows of a: a lane ends up with four consecutive n of one m
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bfrag, afrag, c, SM_FP8_E4M3, FA, OP, sb, OP, sa);
}

// BM x BN output tile per block, waves WM x WN; a stage = one block of 128 along K of both operands, double-buffered in
// LDS and filled by direct loads (16 bytes per lane, no registers). LDS rows are 128 bytes; the 16-byte chunk c of row r
// sits at chunk c ^ (r & 7), so that the eight lanes of a read phase hit eight different chunk columns. A lane's 32 bytes of
// an operand row are chunks g and g + 4 (g = lane / 16): the same permutation of k on both sides leaves the sum as it is,
// and a block of 128 has ONE scale, so it does not matter which quarter a lane holds.
template <int BM, int BN, int WM, int WN, int FA, bool F32S, bool NATIVE>
__global__ __launch_bounds__(WM* WN * 64) void fp8_matmul_kernel(MatmulArgs g) {
    constexpr int NT = WM * WN * 64;
    constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    __shared__ __align__(16) uint8_t lds[2][(BM + BN) * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const int mt = (g.M + BM - 1) / BM, nt = (g.N + BN - 1) / BN;
    // XCD-contiguous shares of the tiles, walked in groups of 8 rows of tiles: the blocks of an XCD share operand rows in its L2
    const int id = xcd_linear(blockIdx.x, mt * nt);
    const int group = id / (8 * nt), gm = min(8, mt - group * 8), in = id - group * 8 * nt;
    const int m0 = (group * 8 + in % gm) * BM, n0 = in / gm * BN;
    const int kb0 = blockIdx.y * g.kb_per_split, kb1 = min(g.KB, kb0 + g.kb_per_split);

    // one direct load moves 64 lanes x 16 bytes = 8 rows; lane i's data lands at byte 16 i of the wave's kilobyte
    constexpr int NL = (BM + BN) * 128 / (NT * 16);
    const uint8_t* src[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int rowbase = (i * (NT / 64) + wave) * 8, r8 = lane >> 3, c = (lane & 7) ^ r8;      // rowbase: wave-uniform
        src[i] = (rowbase < BM ? g.a + (size_t)min(m0 + rowbase + r8, g.M - 1) * g.a_pitch
                               : g.b + (size_t)min(n0 + rowbase - BM + r8, g.N - 1) * g.b_pitch) + (size_t)kb0 * 128 + c * 16;
    }
    auto stage = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src[i],
                                             (__attribute__((address_space(3))) void*)(lds[buf] + (i * (NT / 64) + wave) * 1024), 16, 0, 0);
            src[i] += 128;
        }
    };
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int lr = lane & 15, lg = lane >> 4;
    int arow[TM], brow[TN];      // scale rows of this lane
#pragma unroll
    for (int j = 0; j < TM; ++j) arow[j] = min(m0 + (wm * TM + j) * 16 + lr, g.M - 1);
#pragma unroll
    for (int i = 0; i < TN; ++i) brow[i] = min(n0 + (wn * TN + i) * 16 + lr, g.N - 1) >> g.b_shift;

    int sa[TM], sb[TN];
    auto load_scales = [&](int kq) {
        const uint32_t* pa = static_cast<const uint32_t*>(g.as) + (size_t)kq * g.M;
        const uint32_t* pb = static_cast<const uint32_t*>(g.bs) + (size_t)kq * g.bs_rows;
#pragma unroll
        for (int j = 0; j < TM; ++j) sa[j] = (int)pa[arow[j]];
#pragma unroll
        for (int i = 0; i < TN; ++i) sb[i] = (int)pb[brow[i]];
    };
    auto frag = [&](const uint8_t* base, int row) {
        const u32x4 lo = *reinterpret_cast<const u32x4*>(base + row * 128 + ((lg ^ (row & 7)) << 4));
        const u32x4 hi = *reinterpret_cast<const u32x4*>(base + row * 128 + (((lg + 4) ^ (row & 7)) << 4));
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    // fp32 scales: the block's sum on its own, then one multiply-add per element with sa[m] sb[n]
    f32x4 fb[TN];
    float fa[TM];
    auto block_scales = [&](int kb) {
        const float* pa = static_cast<const float*>(g.as) + (size_t)kb * g.M;
        const float* pb = static_cast<const float*>(g.bs) + (size_t)kb * g.bs_rows;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) fb[i][e] = pb[min(n0 + (wn * TN + i) * 16 + lg * 4 + e, g.N - 1) >> g.b_shift];
#pragma unroll
        for (int j = 0; j < TM; ++j) fa[j] = pa[arow[j]];
    };
    auto add_block = [&](f32x4& c, f32x4 d, float sam, f32x4 sbn) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = fmaf(d[e], sam * sbn[e], c[e]);
    };
    auto compute = [&](auto opc, int buf, int kb) {
        constexpr int OP = decltype(opc)::value;
        const uint8_t* la = lds[buf];
        const uint8_t* lb = la + BM * 128;
        if constexpr (NATIVE) {
            i32x8 bf[TN];
#pragma unroll
            for (int i = 0; i < TN; ++i) bf[i] = frag(lb, (wn * TN + i) * 16 + lr);
            if constexpr (!F32S) {
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    const i32x8 af = frag(la, (wm * TM + j) * 16 + lr);
#pragma unroll
                    for (int i = 0; i < TN; ++i) acc[i][j] = mfma_block<OP, FA>(bf[i], af, acc[i][j], sb[i], sa[j]);
                }
            } else {
                block_scales(kb);
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    const i32x8 af = frag(la, (wm * TM + j) * 16 + lr);
#pragma unroll
                    for (int i = 0; i < TN; ++i)
                        add_block(acc[i][j], mfma_block<0, FA>(bf[i], af, f32x4{0.f, 0.f, 0.f, 0.f}, 0x7f7f7f7f, 0x7f7f7f7f), fa[j], fb[i]);
                }
            }
        } else {
            Wide bw[TN];
#pragma unroll
            for (int i = 0; i < TN; ++i)
                bw[i] = widen<SM_FP8_E4M3>(frag(lb, (wn * TN + i) * 16 + lr), F32S ? 1.f : byte_scale<OP>(sb[i]));
            if constexpr (F32S) block_scales(kb);
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                const Wide aw = widen<FA>(frag(la, (wm * TM + j) * 16 + lr), F32S ? 1.f : byte_scale<OP>(sa[j]));
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    if constexpr (F32S) add_block(acc[i][j], mfma_wide(bw[i], aw, f32x4{0.f, 0.f, 0.f, 0.f}), fa[j], fb[i]);
                    else acc[i][j] = mfma_wide(bw[i], aw, acc[i][j]);
                }
            }
        }
    };
    if (kb0 < kb1) {
        stage(0);
        if constexpr (!F32S) load_scales(kb0 >> 2);
        wait_loads();
        __syncthreads();
        int buf = 0;
        // kb0 is a multiple of 4: block kb's scale byte is byte kb % 4 of its dword, a constant of the unrolled step
        for (int kb = kb0; kb < kb1; kb += 4) {
            auto step = [&](auto opc) {
                const int k = kb + decltype(opc)::value;
                if (k >= kb1) return;
                if (k + 1 < kb1) stage(buf ^ 1);
                compute(opc, buf, k);
                if (decltype(opc)::value == 3 && !F32S && k + 1 < kb1) load_scales((k + 1) >> 2);
                wait_loads();
                __syncthreads();
                buf ^= 1;
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
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

struct Plan {
    int bm, bn, splits, kb_per_split;
};
static Plan matmul_plan(int M, int N, int KB) {
    Plan p{128, 128, 1, KB};
    return p;
}

template <int BM, int BN, int WM, int WN, bool NATIVE>
static void launch_matmul(const MatmulArgs& g, int a_fmt, bool f32s, int splits, hipStream_t s) {
    const dim3 grid((unsigned)(((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN)), (unsigned)splits), block(WM * WN * 64);
    if (f32s) {
        if (a_fmt == SM_FP8_E4M3) hipLaunchKernelGGL((fp8_matmul_kernel<BM, BN, WM, WN, 0, true, NATIVE>), grid, block, 0, s, g);
        else hipLaunchKernelGGL((fp8_matmul_kernel<BM, BN, WM, WN, 1, true, NATIVE>), grid, block, 0, s, g);
    } else {
        if (a_fmt == SM_FP8_E4M3) hipLaunchKernelGGL((fp8_matmul_kernel<BM, BN, WM, WN, 0, false, NATIVE>), grid, block, 0, s, g);
        else hipLaunchKernelGGL((fp8_matmul_kernel<BM, BN, WM, WN, 1, false, NATIVE>), grid, block, 0, s, g);
    }
}

template <int T>
static int launch_quantize(const QuantArgs& a, int tiles, hipStream_t s) {
    const dim3 grid((unsigned)((a.cols + 127) / 128), (unsigned)((a.rows + 127) / 128));
    const bool q = a.q != nullptr, qt = a.qt != nullptr;
    if (tiles) {
        if (q && qt) hipLaunchKernelGGL((fp8_quantize_kernel<T, true, true, true>), grid, dim3(256), 0, s, a);
        else if (q) hipLaunchKernelGGL((fp8_quantize_kernel<T, true, true, false>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((fp8_quantize_kernel<T, true, false, true>), grid, dim3(256), 0, s, a);
    } else {
        if (q && qt) hipLaunchKernelGGL((fp8_quantize_kernel<T, false, true, true>), grid, dim3(256), 0, s, a);
        else if (q) hipLaunchKernelGGL((fp8_quantize_kernel<T, false, true, false>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((fp8_quantize_kernel<T, false, false, true>), grid, dim3(256), 0, s, a);
    }
    SM_LAUNCH_CHECK();
    return 0;
}

}  // namespace sm

extern "C" {

int sm_fp8_quantize(const void* x, int x_type, int rows, int cols, size_t x_stride, int fmt, int tiles, void* q, void* q_scale,
                    void* qt, void* qt_scale, void* stream) {
    if (rows < 0 || cols < 0 || x_type < 0 || x_type > SM_TYPE_F16 || (fmt != SM_FP8_E4M3 && fmt != SM_FP8_E5M2) ||
        (q == nullptr) != (q_scale == nullptr) || (qt == nullptr) != (qt_scale == nullptr) || (q == nullptr && qt == nullptr))
        return (int)hipErrorInvalidValue;
    if (rows == 0 || cols == 0) return 0;
    if (x == nullptr || x_stride < (size_t)cols || (rows + 127) / 128 > 65535) return (int)hipErrorInvalidValue;
    const sm::QuantArgs a{x, x_stride, rows, cols, fmt, (uint8_t*)q, (uint8_t*)q_scale, (uint8_t*)qt, (uint8_t*)qt_scale};
    hipStream_t s = (hipStream_t)stream;
    if (x_type == SM_TYPE_F32) return sm::launch_quantize<SM_TYPE_F32>(a, tiles, s);
    if (x_type == SM_TYPE_BF16) return sm::launch_quantize<SM_TYPE_BF16>(a, tiles, s);
    return sm::launch_quantize<SM_TYPE_F16>(a, tiles, s);
}

size_t sm_fp8_matmul_ws_bytes(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const sm::Plan p = sm::matmul_plan(M, N, (K + 127) / 128);
    return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) : 0;
}

int sm_fp8_matmul(const void* a, const void* a_scale, int a_fmt, size_t a_pitch, const void* b, const void* b_scale, int b_tiles,
                  size_t b_pitch, int scale_f32, int M, int N, int K, void* out, int out_type, size_t out_stride, int accumulate,
                  void* ws, size_t ws_bytes, void* stream) {
    if (M < 0 || N < 0 || K < 0 || out_type < 0 || out_type > SM_TYPE_F16 || (a_fmt != SM_FP8_E4M3 && a_fmt != SM_FP8_E5M2))
        return (int)hipErrorInvalidValue;
    if (M == 0 || N == 0) return 0;
    if (out == nullptr || out_stride < (size_t)N) return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    const int KB = (K + 127) / 128;
    sm::MatmulArgs g{(const uint8_t*)a, (const uint8_t*)b, a_scale, b_scale, out, (float*)ws, a_pitch, b_pitch, out_stride, M, N, KB,
                     b_tiles ? 7 : 0, b_tiles ? (N + 127) / 128 : N, out_type, accumulate, KB};
    const size_t quads = (size_t)(N + 3) / 4 * M;
    if (K == 0) {
        if (!accumulate) hipLaunchKernelGGL(sm::fp8_matmul_empty_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, g);
        SM_LAUNCH_CHECK();
        return 0;
    }
    if (a == nullptr || b == nullptr || a_scale == nullptr || b_scale == nullptr || a_pitch < (size_t)KB * 128 ||
        b_pitch < (size_t)KB * 128 || a_pitch % 16 || b_pitch % 16 || (uintptr_t)a % 16 || (uintptr_t)b % 16)
        return (int)hipErrorInvalidValue;
    const sm::Plan p = sm::matmul_plan(M, N, KB);
    if (p.splits > 1 && (ws == nullptr || ws_bytes < (size_t)p.splits * M * N * sizeof(float))) return (int)hipErrorInvalidValue;
    g.kb_per_split = p.kb_per_split;
    sm::launch_matmul<128, 128, 2, 2, false>(g, a_fmt, scale_f32 != 0, p.splits, s);
    SM_LAUNCH_CHECK();
    if (p.splits > 1) {
        hipLaunchKernelGGL(sm::fp8_matmul_reduce_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, g, p.splits);
        SM_LAUNCH_CHECK();
    }
    return 0;
}

}  // extern "C"
