// The global gradient norm over many tensors and clipping by it, for gfx950.
//
//   norm_2 = s * sqrt(sum g^2), norm_inf = s * max |g|, coefficient = s * min(1, max_norm / (norm + 1e-6)), out = round(g * c)
//
// Both are bound by HBM: the norm reads every gradient once, the clip reads it again and writes it.  One workgroup takes one
// piece of at most 16384 elements of one tensor and leaves one 64-bit partial; a fold of the partials in a fixed order
// gives the norm (no atomics, so the same gradients give the same bits).  Squares are added in 64 bits: fp32 squares are
// exact there and can neither overflow nor vanish.

#include "wq_grad_common.h"

namespace wq {

// Both kernels: a workgroup takes 16 KiB of a gradient, four 16-byte loads per lane, all issued before the first use; an
// unused dynamic LDS allocation caps the workgroups per CU.
constexpr int kLoads = 4;
constexpr int kNormPiecesPerXcdRun = 32;
constexpr unsigned kNormOccupancyPadBytes = 27000;   // 6 workgroups per CU
constexpr int kScalePiecesPerXcdRun = 32;
constexpr unsigned kScaleOccupancyPadBytes = 54000;  // 3

// ---- norm of a piece ------------------------------------------------------------------------------------------------
template <int NORM, int D>
__device__ __forceinline__ void add_vec(typename NormAcc<NORM>::T& a, u32x4 v)
{
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (D == WQ_DTYPE_F32) {
            NormAcc<NORM>::add(a, u2f(v[k]));
        } else {
            const f32x2 f = unpack2<D>(v[k]);
            NormAcc<NORM>::add(a, f.x);
            NormAcc<NORM>::add(a, f.y);
        }
    }
}
template <int NORM, int D>
__device__ __forceinline__ typename NormAcc<NORM>::T piece_norm(const GradPiece& p)
{
    constexpr int kVec = 16 / dtype_bytes(D), kBatch = kLoads * kGradThreads;
    typename NormAcc<NORM>::T a = NormAcc<NORM>::zero();
    const int t = threadIdx.x, head = head_of(p.g, dtype_bytes(D), p.n), whole = (p.n - head) / kVec;
    const char* g = p.g + head * dtype_bytes(D);
    for (int b = 0; b < whole; b += kBatch) {
        u32x4 v[kLoads];
        if (b + kBatch <= whole) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) v[i] = ldg16_nt(g + (size_t)(b + i * kGradThreads + t) * 16);
        } else {  // lanes past the end load the last vector and count it as zeros
#pragma unroll
            for (int i = 0; i < kLoads; ++i) v[i] = ldg16_nt(g + (size_t)min(b + i * kGradThreads + t, whole - 1) * 16);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (b + i * kGradThreads + t >= whole) v[i] = (u32x4){0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) add_vec<NORM, D>(a, v[i]);
    }
    if (t < head) NormAcc<NORM>::add(a, load_elem<D>(p.g, t));
    const int e = whole * kVec + t;
    if (e < p.n - head) NormAcc<NORM>::add(a, load_elem<D>(g, e));
    return a;
}

template <int NORM, typename Source>
__global__ __launch_bounds__(kGradThreads) void grad_norm_partials_kernel(const Source src, const int64_t n_items, char* partials)
{
    typedef typename NormAcc<NORM>::T T;
    __shared__ T lds[kGradThreads / 64];
    const int64_t slot = (int64_t)blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
    if (slot >= n_items) return;  // uniform per workgroup
    const int64_t item = xcd_chunked_item(slot, n_items, kNormPiecesPerXcdRun);
    const GradPiece p = src.piece(item);
    T a;
    if (p.g_dtype == WQ_DTYPE_BF16) a = piece_norm<NORM, WQ_DTYPE_BF16>(p);
    else if (p.g_dtype == WQ_DTYPE_F16) a = piece_norm<NORM, WQ_DTYPE_F16>(p);
    else a = piece_norm<NORM, WQ_DTYPE_F32>(p);
    a = block_fold<NORM, kGradThreads / 64>(a, lds);
    if (threadIdx.x == 0) stg<T>(partials + item * 8, a);
}

// one workgroup per kFoldGroup partials
template <int NORM>
__global__ __launch_bounds__(kGradThreads) void grad_norm_fold_kernel(const char* partials, const int64_t n, char* sums)
{
    typedef typename NormAcc<NORM>::T T;
    __shared__ T lds[kGradThreads / 64];
    const int64_t from = (int64_t)blockIdx.x * kFoldGroup, left = n - from;
    const T a = fold_partials<NORM, kGradThreads>(partials + from * 8, left < kFoldGroup ? left : kFoldGroup, lds);
    if (threadIdx.x == 0) stg<T>(sums + (int64_t)blockIdx.x * 8, a);
}

template <int NORM>
__global__ __launch_bounds__(1024) void grad_norm_total_kernel(const char* partials, const int64_t n, const float scale,
                                                              const float* scale_dev, float* total)
{
    typedef typename NormAcc<NORM>::T T;
    __shared__ T lds[16];
    const T a = fold_partials<NORM, 1024>(partials, n, lds);
    if (threadIdx.x == 0) stg<float>(total, NormAcc<NORM>::finish(a, effective_scale(scale, scale_dev)));
}

// one workgroup per tensor
template <int NORM>
__global__ __launch_bounds__(kGradThreads) void grad_norm_each_kernel(const char* partials, const int64_t* item_start, const float scale,
                                                                     const float* scale_dev, float* each)
{
    typedef typename NormAcc<NORM>::T T;
    __shared__ T lds[kGradThreads / 64];
    const int64_t from = item_start[blockIdx.x], to = item_start[blockIdx.x + 1];
    const T a = fold_partials<NORM, kGradThreads>(partials + from * 8, to - from, lds);
    if (threadIdx.x == 0) stg<float>(each + blockIdx.x, NormAcc<NORM>::finish(a, effective_scale(scale, scale_dev)));
}

// ---- clip of a piece --------------------------------------------------------------------------------------------------
// A lane takes the elements of one 16-byte access of the wider of the two types.
template <int G, int O> struct ScaleVec {
    static constexpr int kElems = G == WQ_DTYPE_F32 || O == WQ_DTYPE_F32 ? 4 : 8;
    static constexpr int kIn = kElems * dtype_bytes(G), kOut = kElems * dtype_bytes(O);
    uint32_t w[kIn / 4];
    __device__ __forceinline__ void load(const char* p)
    {
        if constexpr (kIn == 16) {
            const u32x4 v = ldg16_nt(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const u32x2 v = ldg8_nt(p);
            w[0] = v.x, w[1] = v.y;
        }
    }
    __device__ __forceinline__ void scale_and_store(char* p, float c) const
    {
        float f[kElems];
#pragma unroll
        for (int k = 0; k < kIn / 4; ++k) {
            if constexpr (G == WQ_DTYPE_F32) {
                f[k] = u2f(w[k]) * c;
            } else {
                const f32x2 x = unpack2<G>(w[k]);
                f[2 * k] = x.x * c;
                f[2 * k + 1] = x.y * c;
            }
        }
        if constexpr (O == WQ_DTYPE_F32) stg_nt_sc1<u32x4>(p, (u32x4){f2u(f[0]), f2u(f[1]), f2u(f[2]), f2u(f[3])});
        else if constexpr (kElems == 4) stg_nt_sc1<u32x2>(p, (u32x2){pack2<O>(f[0], f[1]), pack2<O>(f[2], f[3])});
        else stg_nt_sc1<u32x4>(p, (u32x4){pack2<O>(f[0], f[1]), pack2<O>(f[2], f[3]), pack2<O>(f[4], f[5]), pack2<O>(f[6], f[7])});
    }
};
template <int G, int O>
__device__ __forceinline__ void piece_scale(const GradPiece& p, float c)
{
    typedef ScaleVec<G, O> Vec;
    constexpr int kBatch = kLoads * kGradThreads;
    constexpr int kG = dtype_bytes(G), kO = dtype_bytes(O);
    const int t = threadIdx.x, head = kO >= kG ? head_of(p.out, kO, p.n) : head_of(p.g, kG, p.n), n = p.n - head, whole = n / Vec::kElems;
    const char* g = p.g + head * kG;
    char* out = p.out + head * kO;
    for (int b = 0; b < whole; b += kBatch) {
        Vec v[kLoads];
        if (b + kBatch <= whole) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) v[i].load(g + (size_t)(b + i * kGradThreads + t) * Vec::kIn);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) v[i].scale_and_store(out + (size_t)(b + i * kGradThreads + t) * Vec::kOut, c);
        } else {  // lanes past the end load the last vector (in place perhaps as its owner stores it) and drop it
#pragma unroll
            for (int i = 0; i < kLoads; ++i) v[i].load(g + (size_t)min(b + i * kGradThreads + t, whole - 1) * Vec::kIn);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (b + i * kGradThreads + t < whole) v[i].scale_and_store(out + (size_t)(b + i * kGradThreads + t) * Vec::kOut, c);
        }
    }
    const int e = whole * Vec::kElems + t;
    if (e < n) store_elem<O>(out, e, load_elem<G>(g, e) * c);
    if (t < head) store_elem<O>(p.out, t, load_elem<G>(p.g, t) * c);
}
template <int G>
__device__ __forceinline__ void piece_scale_from(const GradPiece& p, float c)
{
    if (p.out_dtype == WQ_DTYPE_BF16) piece_scale<G, WQ_DTYPE_BF16>(p, c);
    else if (p.out_dtype == WQ_DTYPE_F16) piece_scale<G, WQ_DTYPE_F16>(p, c);
    else piece_scale<G, WQ_DTYPE_F32>(p, c);
}

template <typename Source>
__global__ __launch_bounds__(kGradThreads) void grad_scale_kernel(const Source src, const int64_t n_items, const float* total,
                                                                 const float max_norm, const float scale, const float* scale_dev)
{
    const int64_t slot = (int64_t)blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
    if (slot >= n_items) return;  // uniform per workgroup
    const float c = clip_coefficient(ldg<float>(total), max_norm, effective_scale(scale, scale_dev));
    // last piece first: what the norm read last is what a cache still holds
    const GradPiece p = src.piece(n_items - 1 - xcd_chunked_item(slot, n_items, kScalePiecesPerXcdRun));
    if (c == 1.0f && p.out == p.g) return;
    if (p.g_dtype == WQ_DTYPE_BF16) piece_scale_from<WQ_DTYPE_BF16>(p, c);
    else if (p.g_dtype == WQ_DTYPE_F16) piece_scale_from<WQ_DTYPE_F16>(p, c);
    else piece_scale_from<WQ_DTYPE_F32>(p, c);
}

// ---- per-tensor descriptors -> one per piece ----------------------------------------------------------------------------
// Hides that a per-lane factor is a power of two.  From "times 4096 or 8192" the compiler makes a 64-bit shift by a VGPR, and
// on gfx950 that shift goes wrong now and then if the amount is in the last VGPR the kernel has (100 of 13 863 wavefronts
// left their value unshifted): as a number it multiplies.
__device__ __forceinline__ int plain_factor(int x)
{
    asm("" : "+v"(x));
    return x;
}
__global__ __launch_bounds__(256) void grad_make_items_kernel(const int64_t* descs, const int64_t* __restrict__ item_start,
                                                             const int n_desc, const int64_t n_items, const int words, int64_t* items)
{
    const int64_t t = ((int64_t)blockIdx.x + (int64_t)blockIdx.y * gridDim.x) * 256 + threadIdx.x;
    if (t >= n_items) return;
    int i = 0, hi = n_desc;
    while (hi - i > 1) {  // item_start[i] <= t < item_start[hi]
        const int mid = (i + hi) >> 1;
        if (item_start[mid] <= t) i = mid; else hi = mid;
    }
    const int64_t* d = descs + (int64_t)i * words;
    int64_t* o = items + t * words;
    const int g_dtype = (int)(uint32_t)d[3], out_dtype = (int)(uint32_t)((uint64_t)d[3] >> 32);
    const int g_bytes = plain_factor(dtype_bytes(g_dtype)), out_bytes = plain_factor(dtype_bytes(out_dtype));
    const Run r = words == 4 ? run_of(t - item_start[i], d[2], plain_factor(grad_item(g_dtype)), grad_phase(*(const wq_grad_desc*)d))
                             : run_of(t - item_start[i], d[2], kAdamItem, phase_of((const void*)d[4], 4));
    o[0] = d[0] + r.at * g_bytes;
    o[1] = d[1] ? d[1] + r.at * out_bytes : 0;
    o[2] = r.n;
    o[3] = d[3];
    if (words == 8) {
        o[4] = d[4] + r.at * 4;
        o[5] = d[5] + r.at * 4;
        o[6] = d[6] + r.at * 4;
        o[7] = d[7];
    }
}

template <int NORM, typename Source>
static Partials launch_partials(const Source& src, int64_t n_items, void* workspace, hipStream_t st)
{
    char* partials = partials_of(workspace);
    if (n_items) grad_norm_partials_kernel<NORM><<<grid_for_items(n_items), kGradThreads, kNormOccupancyPadBytes, st>>>(src, n_items, partials);
    if (n_items <= kFoldDirect) return {partials, n_items};
    const int64_t groups = cdiv64(n_items, kFoldGroup);
    char* sums = partials + n_items * 8;
    grad_norm_fold_kernel<NORM><<<(unsigned)groups, kGradThreads, 0, st>>>(partials, n_items, sums);
    return {sums, groups};
}
Partials launch_norm_partials(const TableSource& src, int64_t n_items, int norm, void* workspace, hipStream_t st)
{
    return norm == WQ_NORM_2 ? launch_partials<WQ_NORM_2>(src, n_items, workspace, st) : launch_partials<WQ_NORM_INF>(src, n_items, workspace, st);
}

template <int NORM, typename Source>
static void launch_norm_kind(const Source& src, int64_t n_items, float scale, const float* scale_dev, void* workspace, float* total,
                             hipStream_t st)
{
    const Partials p = launch_partials<NORM>(src, n_items, workspace, st);
    grad_norm_total_kernel<NORM><<<1, 1024, 0, st>>>(p.at, p.n, scale, scale_dev, total);
}
template <typename Source>
static void launch_norm(const Source& src, int64_t n_items, int norm, float scale, const float* scale_dev, void* workspace,
                        float* total, hipStream_t st)
{
    if (norm == WQ_NORM_2) launch_norm_kind<WQ_NORM_2>(src, n_items, scale, scale_dev, workspace, total, st);
    else launch_norm_kind<WQ_NORM_INF>(src, n_items, scale, scale_dev, workspace, total, st);
}
template <typename Source>
static void launch_clip(const Source& src, int64_t n_items, int norm, float max_norm, float scale, const float* scale_dev,
                        const float* given, void* workspace, float* total, hipStream_t st)
{
    if (!given) launch_norm(src, n_items, norm, scale, scale_dev, workspace, total, st);
    if (n_items == 0) return;
    grad_scale_kernel<<<grid_for_items(n_items), kGradThreads, kScaleOccupancyPadBytes, st>>>(src, n_items, given ? given : total,
                                                                                              max_norm, scale, scale_dev);
}

static bool grad_dtype_ok(int d) { return d == WQ_DTYPE_BF16 || d == WQ_DTYPE_F16 || d == WQ_DTYPE_F32; }

// per-tensor HOST descriptors -> kernel arguments; negative: an error
static int64_t few_source(const wq_grad_desc* descs, int n_desc, bool with_out, FewSource* src)
{
    if (n_desc < 0 || n_desc > WQ_GRAD_FEW_MAX) return WQ_ERR_SHAPE;
    if (n_desc && !descs) return WQ_ERR_NULL;
    int64_t items = 0;
    int k = 0;
    for (int i = 0; i < n_desc; ++i) {
        if (descs[i].n < 0) return WQ_ERR_SHAPE;
        if (!grad_dtype_ok(descs[i].g_dtype) || (with_out && !grad_dtype_ok(descs[i].out_dtype))) return WQ_ERR_MODE;
        if (descs[i].n == 0) continue;
        if (!descs[i].g || (with_out && !descs[i].out)) return WQ_ERR_NULL;
        src->d[k] = descs[i];
        if (!with_out) src->d[k].out = nullptr;
        src->start[k++] = items;
        items += pieces_of(descs[i].n, grad_item(descs[i].g_dtype), grad_phase(src->d[k - 1]));
    }
    src->start[k] = items;
    src->n_desc = k;
    return items;
}

}  // namespace wq

using namespace wq;

WQ_EXPORT int64_t wq_grad_workspace_bytes(int64_t n_items) { return n_items < 0 ? 0 : kGradControlBytes + (n_items + cdiv64(n_items, kFoldGroup)) * 8; }

WQ_EXPORT int wq_grad_make_items(const void* descs, const int64_t* item_start, int n_desc, int64_t n_items, int words, void* items,
                                 void* stream)
{
    if (n_desc < 0 || n_items < 0 || (words != 4 && words != 8)) return WQ_ERR_SHAPE;
    if (n_items == 0) return WQ_OK;
    if (n_desc == 0) return WQ_ERR_SHAPE;
    if (!descs || !item_start || !items) return WQ_ERR_NULL;
    grad_make_items_kernel<<<grid_for_items(cdiv64(n_items, 256)), 256, 0, (hipStream_t)stream>>>(
        (const int64_t*)descs, item_start, n_desc, n_items, words, (int64_t*)items);
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}

WQ_EXPORT int wq_grad_norm_items(const void* items, int64_t n_items, int words, const int64_t* item_start, int n_desc, int norm,
                                 float grad_scale, const float* grad_scale_dev, void* workspace, float* total, float* each,
                                 void* stream)
{
    if (n_items < 0 || n_desc < 0 || (words != 4 && words != 8)) return WQ_ERR_SHAPE;
    if (norm != WQ_NORM_2 && norm != WQ_NORM_INF) return WQ_ERR_MODE;
    if (!workspace || !total || (n_items && !items) || (each && n_desc && !item_start)) return WQ_ERR_NULL;
    hipStream_t st = (hipStream_t)stream;
    launch_norm(TableSource{(const int64_t*)items, words}, n_items, norm, grad_scale, grad_scale_dev, workspace, total, st);
    if (each && n_desc) {
        const char* partials = partials_of(workspace);
        if (norm == WQ_NORM_2) grad_norm_each_kernel<WQ_NORM_2><<<n_desc, kGradThreads, 0, st>>>(partials, item_start, grad_scale, grad_scale_dev, each);
        else grad_norm_each_kernel<WQ_NORM_INF><<<n_desc, kGradThreads, 0, st>>>(partials, item_start, grad_scale, grad_scale_dev, each);
    }
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}

WQ_EXPORT int wq_grad_norm_few(const wq_grad_desc* descs, int n_desc, int norm, float grad_scale, void* workspace, float* total,
                               void* stream)
{
    if (norm != WQ_NORM_2 && norm != WQ_NORM_INF) return WQ_ERR_MODE;
    FewSource src;
    const int64_t items = few_source(descs, n_desc, false, &src);
    if (items < 0) return (int)items;
    if (!workspace || !total) return WQ_ERR_NULL;
    launch_norm(src, items, norm, grad_scale, nullptr, workspace, total, (hipStream_t)stream);
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}

WQ_EXPORT int wq_grad_clip_items(const wq_grad_desc* items, int64_t n_items, int norm, float max_norm, float grad_scale,
                                 const float* grad_scale_dev, const float* total_given, void* workspace, float* total, void* stream)
{
    if (n_items < 0) return WQ_ERR_SHAPE;
    if (norm != WQ_NORM_2 && norm != WQ_NORM_INF) return WQ_ERR_MODE;
    if ((!total_given && (!workspace || !total)) || (n_items && !items)) return WQ_ERR_NULL;
    if (n_items == 0 && total_given) return WQ_OK;
    launch_clip(TableSource{(const int64_t*)items, 4}, n_items, norm, max_norm, grad_scale, grad_scale_dev, total_given, workspace,
                total, (hipStream_t)stream);
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}

WQ_EXPORT int wq_grad_clip_few(const wq_grad_desc* descs, int n_desc, int norm, float max_norm, float grad_scale,
                               const float* total_given, void* workspace, float* total, void* stream)
{
    if (norm != WQ_NORM_2 && norm != WQ_NORM_INF) return WQ_ERR_MODE;
    FewSource src;
    const int64_t items = few_source(descs, n_desc, true, &src);
    if (items < 0) return (int)items;
    if (!total_given && (!workspace || !total)) return WQ_ERR_NULL;
    if (items == 0 && total_given) return WQ_OK;
    launch_clip(src, items, norm, max_norm, grad_scale, nullptr, total_given, workspace, total, (hipStream_t)stream);
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}
