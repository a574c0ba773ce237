// What the gradient norm, the clip and the AdamW update share: element types, piece sources and the fold of the partial
// norms.
#pragma once

#include "wq_common.h"

namespace wq {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kGradThreads = 256;
constexpr int kAdamItem = WQ_ADAMW_ITEM;

// 16- and 8-byte accesses of streams whose elements have their own alignment only (a tensor inside a packed buffer starts
// anywhere): gfx950's global accesses take any address, the type says so to the compiler.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ u32x4 ldg16(const char* p) { return *(const WQ_GLOBAL u32x4_a2*)p; }
__device__ __forceinline__ u32x4 ldg16_nt(const char* p) { return __builtin_nontemporal_load((const WQ_GLOBAL u32x4_a2*)p); }
__device__ __forceinline__ u32x2 ldg8_nt(const char* p) { return __builtin_nontemporal_load((const WQ_GLOBAL u32x2_a2*)p); }

__host__ __device__ constexpr int dtype_bytes(int d) { return d == WQ_DTYPE_F32 ? 4 : 2; }
// elements of a gradient piece
__host__ __device__ constexpr int grad_item(int d) { return WQ_GRAD_ITEM_BYTES / dtype_bytes(d); }

template <int D>
__device__ __forceinline__ float load_elem(const char* p, int i)
{
    if constexpr (D == WQ_DTYPE_F32) return ldg<float>(p + (size_t)i * 4);
    const uint32_t h = ldg<uint16_t>(p + (size_t)i * 2);
    if constexpr (D == WQ_DTYPE_BF16) return u2f(h << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
// two 16-bit elements of a dword
template <int D>
__device__ __forceinline__ f32x2 unpack2(uint32_t w)
{
    if constexpr (D == WQ_DTYPE_BF16) return (f32x2){bf16lo(w), bf16hi(w)};
    return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
}
// One rounding, to nearest even.  The value is pinned to a register first: fused into the multiplication that made it
// (v_fma_mixlo_f16 with a +0 addend) a product of -0 would come out as +0.
template <int D>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    asm("" : "+v"(a));
    asm("" : "+v"(b));
    const f32x2 v = {a, b};
    if constexpr (D == WQ_DTYPE_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <int D>
__device__ __forceinline__ void store_elem(char* p, int i, float v)
{
    if constexpr (D == WQ_DTYPE_F32) stg<float>(p + (size_t)i * 4, v);
    else stg<uint16_t>(p + (size_t)i * 2, (uint16_t)pack2<D>(v, 0.0f));
}

// ---- pieces of a tensor ---------------------------------------------------------------------------------------------
// Pieces are cut where the stream that sets the pace is at a 128-byte line: the first piece of a tensor is shorter by the
// elements between the line before its start and the start (the phase), so that all later ones start on a line and no two
// workgroups write into one line (tensors packed back to back start anywhere: 87 M odd bf16 elements clipped into fp32 took
// 144 us with pieces counted from the start, 125 us so).  The stream is the wider one of a clip, the fp32 weight of an update.
__host__ __device__ __forceinline__ int phase_of(const void* p, int elem_bytes) { return (int)((uintptr_t)p & 127) / elem_bytes; }
__host__ __device__ __forceinline__ int grad_phase(const wq_grad_desc& d)
{
    const int g = dtype_bytes(d.g_dtype), o = dtype_bytes(d.out_dtype);
    return d.out && o >= g ? phase_of(d.out, o) : phase_of(d.g, g);
}
struct Run {
    int64_t at;
    int n;
};
__host__ __device__ __forceinline__ Run run_of(int64_t piece, int64_t n, int item, int phase)
{
    const int64_t from = piece ? piece * item - phase : 0, to = (piece + 1) * item - phase;
    return {from, (int)((to < n ? to : n) - from)};
}
__host__ __device__ __forceinline__ int64_t pieces_of(int64_t n, int item, int phase) { return n ? (n + phase + item - 1) / item : 0; }

// elements before the first 16-byte boundary (a lane each), of at most n
__device__ __forceinline__ int head_of(const char* p, int elem_bytes, int n) { return min((int)(-(uintptr_t)p & 15) / elem_bytes, n); }

// ---- where a workgroup finds its piece ---------------------------------------------------------------------------
struct GradPiece {
    const char* g;
    char* out;
    int n, g_dtype, out_dtype;
};
// A workgroup lives for a few microseconds, and scalar loads that wait for one another (arguments, then the row, then a
// step's scalars ...) are a good part of it: everything a workgroup needs is addressed without a branch and loaded at once -
// a slot behind the last piece reads the last one's row and leaves after that -, and one empty asm that takes all of it keeps
// the compiler from moving a load behind the branches that follow.  WQ_CONST: memory that no one writes while the kernel runs
// (scalar loads).
#define WQ_CONST __attribute__((address_space(4)))
typedef int64_t i64x4 __attribute__((ext_vector_type(4), aligned(8)));
typedef int64_t i64x8 __attribute__((ext_vector_type(8), aligned(8)));
__device__ __forceinline__ uint32_t const_u32(const void* p) { return *(const WQ_CONST uint32_t*)p; }
// the slot's work item (see xcd_chunked_item), without a branch; total > 0
__device__ __forceinline__ int64_t item_of_slot(int64_t slot, int64_t total, int C)
{
    slot = slot < total ? slot : total - 1;
    const int64_t span = (int64_t)kXcds * C, from = slot / span * span;
    const uint32_t r = (uint32_t)(slot - from);
    const int64_t mixed = from + (int64_t)(r % kXcds * C + r / kXcds), whole = -(int64_t)(from + span <= total);
    return (mixed & whole) | (slot & ~whole);
}

// A table with one descriptor per piece; `words` is 4 (wq_grad_desc) or 8 (wq_adamw_desc, which begins alike).
struct TableSource {
    const int64_t* items;
    int words;
    __device__ __forceinline__ GradPiece piece(int64_t t) const
    {
        const i64x4 d = *(const WQ_CONST i64x4*)(items + t * words);
        return {(const char*)d[0], (char*)d[1], (int)d[2], (int)(uint32_t)d[3], (int)((uint64_t)d[3] >> 32)};
    }
};
// Tensors in the kernel arguments (3.5 of their 4 KiB).
struct ListSource {
    const char* g[WQ_GRAD_LIST_LAUNCH];
    uint64_t n_dtype[WQ_GRAD_LIST_LAUNCH];     // elements, type in the top byte
    int32_t start[WQ_GRAD_LIST_LAUNCH];
    int32_t n_tensors;
    __device__ __forceinline__ GradPiece piece(int64_t t) const
    {
        int lo = 0, hi = n_tensors;
        while (hi - lo > 1) {  // start[lo] <= t < start[hi]
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= t) lo = mid; else hi = mid;
        }
        const int dtype = (int)(n_dtype[lo] >> 56), bytes = dtype_bytes(dtype);
        const Run r = run_of(t - start[lo], (int64_t)(n_dtype[lo] & ~(255ull << 56)), grad_item(dtype), phase_of(g[lo], bytes));
        const char* at = g[lo] + r.at * bytes;
        return {at, (char*)at, r.n, dtype, dtype};
    }
};

// ---- partial norms -------------------------------------------------------------------------------------------------
// 2-norm: a partial is a sum of squares (double).  Infinity norm: the largest magnitude's fp32 bits (integers order like
// magnitudes and NaN is above infinity, so a NaN wins), as a uint64.
template <int NORM> struct NormAcc;
template <> struct NormAcc<WQ_NORM_2> {
    typedef double T;
    static __device__ __forceinline__ T zero() { return 0.0; }
    static __device__ __forceinline__ T join(T a, T b) { return a + b; }
    static __device__ __forceinline__ void add(T& a, float x)
    {
        const double d = (double)x;
        a = __builtin_fma(d, d, a);
    }
    static __device__ __forceinline__ float finish(T a, float scale) { return (float)(__builtin_sqrt(a) * (double)__builtin_fabsf(scale)); }
};
template <> struct NormAcc<WQ_NORM_INF> {
    typedef uint64_t T;
    static __device__ __forceinline__ T zero() { return 0; }
    static __device__ __forceinline__ T join(T a, T b) { return a > b ? a : b; }
    static __device__ __forceinline__ void add(T& a, float x) { a = (uint64_t)max((uint32_t)a, f2u(x) & 0x7FFFFFFFu); }
    // without a sign, also where infinity times 0 makes a NaN (with a sign, here): bits order like norms
    static __device__ __forceinline__ float finish(T a, float scale) { return __builtin_fabsf(u2f((uint32_t)a) * scale); }
};

template <typename T>
__device__ __forceinline__ T shfl_xor_64(T v, int m)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, m), hi = (uint32_t)__shfl_xor((int)(uint32_t)(b >> 32), m);
    return __builtin_bit_cast(T, ((uint64_t)hi << 32) | lo);
}
template <int NORM>
__device__ __forceinline__ typename NormAcc<NORM>::T wave_fold(typename NormAcc<NORM>::T a)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) a = NormAcc<NORM>::join(a, shfl_xor_64(a, m));
    return a;
}
// The fold over a workgroup of WAVES wavefronts; valid in every lane.  lds: WAVES values.
template <int NORM, int WAVES>
__device__ __forceinline__ typename NormAcc<NORM>::T block_fold(typename NormAcc<NORM>::T a, typename NormAcc<NORM>::T* lds)
{
    a = wave_fold<NORM>(a);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    a = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) a = NormAcc<NORM>::join(a, lds[w]);
    return a;
}

// The fold of n values by one workgroup of THREADS, in an order that depends on n only; four loads in flight per lane (8: +0.7,
// 16: +0.7 us on 12 300 values).
template <int NORM, int THREADS>
__device__ __forceinline__ typename NormAcc<NORM>::T fold_partials(const char* partials, int64_t n, typename NormAcc<NORM>::T* lds)
{
    typedef typename NormAcc<NORM>::T T;
    T a = NormAcc<NORM>::zero();
    for (int64_t i = threadIdx.x; i < n; i += 4 * THREADS) {
        T v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t k = i + u * THREADS;
            v[u] = ldg<T>(partials + (k < n ? k : n - 1) * 8);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * THREADS < n) a = NormAcc<NORM>::join(a, v[u]);
    }
    return block_fold<NORM, THREADS / 64>(a, lds);
}

__device__ __forceinline__ float effective_scale(float scale, const float* dev) { return dev ? scale * ldg<float>(dev) : scale; }
__device__ __forceinline__ float clip_coefficient(float norm, float max_norm, float scale)
{
    const float c = max_norm / (norm + 1e-6f);
    return (c > 1.0f ? 1.0f : c) * scale;      // NaN stays NaN
}

// workspace: 64 bytes of AdamW's per-step values, one partial per piece, and the sums of kFoldGroup partials each that long
// lists fold first (norms of 17 280 pieces 44.8 us in one fold, 45.9 in two; of 27 648 68.2 and 68.6; of 32 640 79.2 and 79.3; of 36 864
// 88.4 and 88.1; of 55 296 130.4 and 127.9; of 110 592 260 and 247).
constexpr int64_t kGradControlBytes = 64;
constexpr int64_t kFoldGroup = 4096, kFoldDirect = 8 * kFoldGroup;
inline char* partials_of(void* workspace) { return (char*)workspace + kGradControlBytes; }
struct Partials {
    const char* at;
    int64_t n;
};

// wq_grad.hip: one partial per piece of an update's table (whose gradients are read again right behind), for more than
// kFoldDirect pieces folded to one value per kFoldGroup
Partials launch_norm_partials(const TableSource& src, int64_t n_items, int norm, void* workspace, hipStream_t st);

}  // namespace wq
