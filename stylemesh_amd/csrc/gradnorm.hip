// G1: the global norm over a list of gradient tensors and clipping by it (include/stylemesh_hip.h section G1): what
// pytorch_lightning's Trainer(gradient_clip_val=...) asks of torch.nn.utils.clip_grad_norm_ between backward and the
// optimizer step.
//
//   norm = sqrt(sum over all tensors of g^2)  or  max |g|        coef = min(1, max_norm / (norm + 1e-6))        out = g coef
//
// Two kernels per 200 tensors: per-block partial sums, then the scaling pass, whose every block adds the same partial sums in
// the same order (a few KB from L2) instead of waiting for a third launch. No atomics: the norm has the same bits every time.
// Sums are held in 64 bits: squares of fp32 gradients over- and underflow fp32 (|g| > 1.8e19, < 1e-23) where the norm
// does not, and the 64-bit multiply-add runs at the fp32 rate on this chip - both kernels are bound by HBM.
#include <cmath>
#include <type_traits>

#include "common.h"

namespace sm {

typedef unsigned g_u32x4 __attribute__((ext_vector_type(4)));
typedef g_u32x4 g_u32x4_u __attribute__((aligned(2)));      // gradient views start at any element
typedef unsigned g_u32x2 __attribute__((ext_vector_type(2)));
typedef g_u32x2 g_u32x2_u __attribute__((aligned(2)));

// tensors per launch: the table travels in the kernel arguments (4 KB; no device copy to keep alive), 20 bytes a tensor. With 32
// bytes and 120 tensors a list of 161 takes four launches instead of two (99 991 bf16 elements each: 35 -> 24 us).
constexpr int GN_TENSORS = 200;
constexpr int GN_PARTIALS = 1024;    // at most this many partial sums per call and launch

struct GradTable {
    unsigned in_lo[GN_TENSORS], out_lo[GN_TENSORS];
    unsigned hi[GN_TENSORS];         // bits 32 ... 47 of in and, above them, of out: device addresses have 48 bits
    unsigned tail[GN_TENSORS];       // elements of the last chunk | SM_TYPE_* of in << 16 | of out << 20
    int first[GN_TENSORS + 1];       // first chunk of each tensor
    int count;
    int chunk_log2;                  // elements per chunk, at most 2^13
};
static_assert(sizeof(GradTable) <= 4096 - 48, "with the kernels' other arguments within 4 KB");

// chunk c of the table's tensors
struct Chunk {
    const void* in;
    void* out;
    size_t begin, end;               // elements of the tensor
    unsigned in_type, out_type;
};

__device__ __forceinline__ double gn_combine(double a, double b, bool inf) {
    if (!inf) return a + b;
    return (b > a || b != b) ? b : a;      // a NaN stays
}
template <bool INF>
__device__ __forceinline__ double gn_take(double acc, float v) {
    if constexpr (!INF) return fma((double)v, (double)v, acc);
    else return gn_combine(acc, (double)fabsf(v), true);
}
// f(type as a constant), chosen once per chunk: the loops inside have no branch left
template <class F>
__device__ __forceinline__ void gn_typed(unsigned type, F f) {
    if (type == SM_TYPE_F32) f(std::integral_constant<int, SM_TYPE_F32>{});
    else if (type == SM_TYPE_BF16) f(std::integral_constant<int, SM_TYPE_BF16>{});
    else f(std::integral_constant<int, SM_TYPE_F16>{});
}
__device__ __forceinline__ double gn_block(double v, bool inf) {
    __shared__ double red[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = gn_combine(v, __shfl_xor(v, o, 64), inf);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return gn_combine(gn_combine(red[0], red[1], inf), gn_combine(red[2], red[3], inf), inf);
}
__device__ __forceinline__ float gn_up(unsigned h, int type) {
    return type == SM_TYPE_BF16 ? __builtin_bit_cast(float, h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
__device__ __forceinline__ unsigned gn_down(float f, int type) {
    if (type == SM_TYPE_F16) return __builtin_bit_cast(uint16_t, (_Float16)f);
    const unsigned u = __builtin_bit_cast(unsigned, f);
    return (u & 0x7fffffffu) > 0x7f800000u ? ((u >> 16) | 0x40u) : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
// elements i ... i + 7 of a tensor as they are, and as fp32
template <int T>
struct Raw8 {
    g_u32x4 d[T == SM_TYPE_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* p, size_t i) {
        const g_u32x4_u* q = reinterpret_cast<const g_u32x4_u*>(static_cast<const char*>(p) + i * (T == SM_TYPE_F32 ? 4 : 2));
        d[0] = q[0];
        if constexpr (T == SM_TYPE_F32) d[1] = q[1];
    }
    __device__ __forceinline__ void get(float* v) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (T == SM_TYPE_F32) {
                v[j] = __builtin_bit_cast(float, (unsigned)d[0][j]);
                v[4 + j] = __builtin_bit_cast(float, (unsigned)d[1][j]);
            } else {
                v[2 * j] = gn_up(d[0][j] & 0xffffu, T);
                v[2 * j + 1] = gn_up(d[0][j] >> 16, T);
            }
        }
    }
};
__device__ __forceinline__ float gn_load1(const void* p, size_t i, int type) {
    return type == SM_TYPE_F32 ? static_cast<const float*>(p)[i] : gn_up(static_cast<const uint16_t*>(p)[i], type);
}
template <int O>
__device__ __forceinline__ void gn_store8(void* p, size_t i, const float* v, bool past) {
    g_u32x4_u* o = reinterpret_cast<g_u32x4_u*>(static_cast<char*>(p) + i * (O == SM_TYPE_F32 ? 4 : 2));
    g_u32x4 a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (O == SM_TYPE_F32) {
            a[j] = __builtin_bit_cast(unsigned, v[j]);
            b[j] = __builtin_bit_cast(unsigned, v[4 + j]);
        } else {
            a[j] = gn_down(v[2 * j], O) | (gn_down(v[2 * j + 1], O) << 16);
        }
    }
    if (past) {
        __builtin_nontemporal_store(a, o);
        if constexpr (O == SM_TYPE_F32) __builtin_nontemporal_store(b, o + 1);
    } else {
        o[0] = a;
        if constexpr (O == SM_TYPE_F32) o[1] = b;
    }
}
__device__ __forceinline__ int gn_tensor_of(const GradTable& t, int chunk) {
    int lo = 0, hi = t.count;              // last tensor with first <= chunk (an empty tensor has no chunk)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ Chunk gn_chunk(const GradTable& t, int c) {
    const int k = gn_tensor_of(t, c);
    const unsigned hi = t.hi[k], tail = t.tail[k];
    Chunk r;
    r.in = reinterpret_cast<const void*>((unsigned long long)t.in_lo[k] | (unsigned long long)(hi & 0xffffu) << 32);
    r.out = reinterpret_cast<void*>((unsigned long long)t.out_lo[k] | (unsigned long long)(hi >> 16) << 32);
    r.begin = (size_t)(c - t.first[k]) << t.chunk_log2;
    r.end = r.begin + (c + 1 == t.first[k + 1] ? tail & 0xffffu : 1u << t.chunk_log2);
    r.in_type = tail >> 16 & 15u;
    r.out_type = tail >> 20;
    return r;
}

template <bool INF>
__global__ __launch_bounds__(256) void grad_norm_partial_kernel(GradTable t, double* __restrict__ partial) {
    double acc = 0.0;
    for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const Chunk k = gn_chunk(t, c);
        const void* in = k.in;
        const size_t end = k.end;
        gn_typed(k.in_type, [&](auto tc) {
            constexpr int T = decltype(tc)::value;
            size_t i = k.begin + threadIdx.x * 8;
            // four rounds of loads in flight
            for (; i + 3 * 2048 + 8 <= end; i += 4 * 2048) {
                Raw8<T> r[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) r[u].load(in, i + u * 2048);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float v[8];
                    r[u].get(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc = gn_take<INF>(acc, v[j]);
                }
            }
            for (; i + 8 <= end; i += 2048) {
                Raw8<T> r;
                float v[8];
                r.load(in, i);
                r.get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) acc = gn_take<INF>(acc, v[j]);
            }
            for (; i < end; ++i) acc = gn_take<INF>(acc, gn_load1(in, i, T));      // (only the thread the end falls to)
        });
    }
    acc = gn_block(acc, INF);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__device__ __forceinline__ double gn_total(const double* partial, int n, bool inf) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) acc = gn_combine(acc, partial[i], inf);
    acc = gn_block(acc, inf);
    return inf ? acc : sqrt(acc);
}

__global__ __launch_bounds__(256) void grad_norm_final_kernel(const double* __restrict__ partial, int n, int inf, float* norm_out) {
    const double norm = gn_total(partial, n, inf != 0);
    if (threadIdx.x == 0) *norm_out = (float)norm;
}

__global__ __launch_bounds__(256) void grad_clip_kernel(GradTable t, const double* __restrict__ partial, int n_partial, int inf,
                                                        double max_norm, int in_place, float* norm_out) {
    const double norm = gn_total(partial, n_partial, inf != 0);
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const double q = max_norm / (norm + 1e-6);
    const float coef = q > 1.0 ? 1.f : (float)q;          // a NaN norm stays NaN, as in the arithmetic it stands for
    if (in_place && coef == 1.f) return;                   // x 1 in place is what is there
    // from the last chunk backwards: the norm's pass ended there, and what it read last may still be in the 256 MB cache
    for (int c = t.first[t.count] - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
        const Chunk k = gn_chunk(t, c);
        const void* in = k.in;
        void* out = k.out;
        const size_t end = k.end;
        gn_typed(k.in_type, [&](auto tc) {
            constexpr int T = decltype(tc)::value;
            gn_typed(k.out_type, [&](auto oc) {
                constexpr int O = decltype(oc)::value;
                size_t i = k.begin + threadIdx.x * 8;
                for (; i + 2048 + 8 <= end; i += 2 * 2048) {
                    Raw8<T> r[2];
                    r[0].load(in, i);
                    r[1].load(in, i + 2048);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float v[8];
                        r[u].get(v);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] *= coef;
                        gn_store8<O>(out, i + u * 2048, v, !in_place);
                    }
                }
                for (; i + 8 <= end; i += 2048) {
                    Raw8<T> r;
                    float v[8];
                    r.load(in, i);
                    r.get(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= coef;
                    gn_store8<O>(out, i, v, !in_place);
                }
                for (; i < end; ++i) {
                    const float x = gn_load1(in, i, T) * coef;
                    if constexpr (O == SM_TYPE_F32) static_cast<float*>(out)[i] = x;
                    else static_cast<uint16_t*>(out)[i] = (uint16_t)gn_down(x, O);
                }
            });
        });
    }
}

}  // namespace sm

namespace {

// chunks of 4096 elements (two rounds of a block's 8-element loads) for short lists, 8192 for long ones (a call's 2^40 elements
// are 2^27 chunks)
int chunk_log2_of(unsigned long long total) { return total >= (8ull << 20) ? 13 : 12; }

// table of tensors [first, first + count) of a call; returns its chunks
int fill_table(sm::GradTable& t, const void* const* in, void* const* out, const size_t* numel, const int* types, const int* out_types,
               int first, int count, int chunk_log2) {
    t.count = count;
    t.chunk_log2 = chunk_log2;
    t.first[0] = 0;
    for (int i = 0; i < count; ++i) {
        const size_t n = numel[first + i];
        const int chunks = (int)((n + ((size_t)1 << chunk_log2) - 1) >> chunk_log2);
        const uint64_t a = n ? (uint64_t)in[first + i] : 0, b = n && out != nullptr ? (uint64_t)out[first + i] : 0;
        const int ty = types[first + i], oty = out_types == nullptr ? ty : out_types[first + i];
        t.in_lo[i] = (unsigned)a;
        t.out_lo[i] = (unsigned)b;
        t.hi[i] = (unsigned)(a >> 32) | (unsigned)(b >> 32) << 16;
        t.tail[i] = chunks ? (unsigned)(n - ((size_t)(chunks - 1) << chunk_log2)) | (unsigned)ty << 16 | (unsigned)oty << 20 : 0;
        t.first[i + 1] = t.first[i] + chunks;
    }
    return t.first[count];
}

int check_list(const void* const* in, const size_t* numel, const int* types, int n, unsigned long long* total) {
    *total = 0;
    if (n < 0 || (n > 0 && (in == nullptr || numel == nullptr || types == nullptr))) return (int)hipErrorInvalidValue;
    for (int i = 0; i < n; ++i) {
        if (types[i] < 0 || types[i] > SM_TYPE_F16 || (numel[i] > 0 && (in[i] == nullptr || (uint64_t)in[i] >> 48 != 0 || numel[i] >> 40)))
            return (int)hipErrorInvalidValue;
        *total += numel[i];
    }
    return *total >> 40 ? (int)hipErrorInvalidValue : 0;
}

// partial sums of every launch of the call into ws; *n_partial = their number
int launch_partials(const void* const* grads, const size_t* numel, const int* types, int n, int inf, int chunk_log2, double* ws,
                    size_t ws_doubles, int* n_partial, hipStream_t s) {
    *n_partial = 0;
    for (int f = 0; f < n; f += sm::GN_TENSORS) {
        sm::GradTable t;
        const int chunks = fill_table(t, grads, nullptr, numel, types, nullptr, f, n - f < sm::GN_TENSORS ? n - f : sm::GN_TENSORS, chunk_log2);
        if (chunks == 0) continue;
        const int blocks = chunks < sm::GN_PARTIALS ? chunks : sm::GN_PARTIALS;
        if ((size_t)(*n_partial + blocks) > ws_doubles) return (int)hipErrorInvalidValue;
        if (inf) hipLaunchKernelGGL(sm::grad_norm_partial_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, s, t, ws + *n_partial);
        else hipLaunchKernelGGL(sm::grad_norm_partial_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, s, t, ws + *n_partial);
        SM_LAUNCH_CHECK();
        *n_partial += blocks;
    }
    return 0;
}

}  // namespace

extern "C" {

size_t sm_grad_norm_ws_bytes(int n_tensors) {
    const int launches = n_tensors <= 0 ? 1 : (n_tensors + sm::GN_TENSORS - 1) / sm::GN_TENSORS;
    return (size_t)launches * sm::GN_PARTIALS * sizeof(double);
}

int sm_grad_norm(const void* const* grads, const size_t* numel, const int* types, int n, int inf_norm, void* ws, size_t ws_bytes,
                 float* norm_out, void* stream) {
    unsigned long long total;
    if (const int e = check_list(grads, numel, types, n, &total)) return e;
    if (norm_out == nullptr || ws == nullptr || (uintptr_t)ws % 8) return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    int n_partial = 0;
    if (const int e = launch_partials(grads, numel, types, n, inf_norm, chunk_log2_of(total), (double*)ws, ws_bytes / sizeof(double), &n_partial, s))
        return e;
    hipLaunchKernelGGL(sm::grad_norm_final_kernel, dim3(1), dim3(256), 0, s, (const double*)ws, n_partial, inf_norm, norm_out);
    SM_LAUNCH_CHECK();
    return 0;
}

int sm_grad_clip(const void* const* grads, void* const* out, const size_t* numel, const int* types, const int* out_types, int n,
                 int inf_norm, double max_norm, void* ws, size_t ws_bytes, float* norm_out, void* stream) {
    unsigned long long total;
    if (const int e = check_list(grads, numel, types, n, &total)) return e;
    if (norm_out == nullptr || ws == nullptr || (uintptr_t)ws % 8 || !(max_norm >= 0.0) || (n > 0 && (out == nullptr || out_types == nullptr)))
        return (int)hipErrorInvalidValue;
    int in_place = 1;
    for (int i = 0; i < n; ++i) {
        if (out_types[i] < 0 || out_types[i] > SM_TYPE_F16 || (numel[i] > 0 && (out[i] == nullptr || (uint64_t)out[i] >> 48 != 0))) return (int)hipErrorInvalidValue;
        if (numel[i] == 0) continue;
        if (out[i] != grads[i]) in_place = 0;
        else if (out_types[i] != types[i]) return (int)hipErrorInvalidValue;
    }
    hipStream_t s = (hipStream_t)stream;
    const int cl = chunk_log2_of(total);
    int n_partial = 0;
    if (const int e = launch_partials(grads, numel, types, n, inf_norm, cl, (double*)ws, ws_bytes / sizeof(double), &n_partial, s)) return e;
    bool told = false;
    for (int f = 0; f < n; f += sm::GN_TENSORS) {
        sm::GradTable t;
        const int chunks = fill_table(t, grads, out, numel, types, out_types, f, n - f < sm::GN_TENSORS ? n - f : sm::GN_TENSORS, cl);
        if (chunks == 0) continue;
        const int blocks = chunks < 2048 ? chunks : 2048;
        hipLaunchKernelGGL(sm::grad_clip_kernel, dim3((unsigned)blocks), dim3(256), 0, s, t, (const double*)ws, n_partial, inf_norm,
                           max_norm, in_place, told ? nullptr : norm_out);
        SM_LAUNCH_CHECK();
        told = true;
    }
    if (!told) {      // no element at all: the norm is 0
        hipLaunchKernelGGL(sm::grad_norm_final_kernel, dim3(1), dim3(256), 0, s, (const double*)ws, 0, inf_norm, norm_out);
        SM_LAUNCH_CHECK();
    }
    return 0;
}

}  // extern "C"
