// The global gradient norm over many tensors and clipping by it, for gfx950.
//
//   norm_2 = s * sqrt(sum g^2), norm_inf = s * max |g|, coefficient = s * min(1, max_norm / (norm + 1e-6)), out = round(g * c)
//
// Both are bound by HBM: the norm reads every gradient once, the clip reads it again and writes it.  One workgroup takes one
// piece - 16 KiB of one tensor, in the table of an update the gradients of 8192 elements - and leaves one 64-bit partial; a fold of
// the partials in a fixed order gives the norm (no atomics: the same list at the same addresses gives the same bits; pieces end at
// 128-byte lines, so other starts add in another order).  Squares are added in 64 bits: fp32 squares are
// exact there and can neither overflow nor vanish.

#include "wq_grad_common.h"

namespace wq {

// Norm: a workgroup takes a piece, four 16-byte loads per lane, all issued before the first use; an unused dynamic LDS
// allocation caps the workgroups per CU.  A whole model's 14.5 GB of fp32 (3.6 G elements, 887 000 pieces): 1938 us = 7.5 TB/s
// with 6 workgroups per CU; 8: 2015, 4: 2094, 3: 2499 us.
constexpr int kNormLoads = 4;
constexpr int kNormPiecesPerXcdRun = 32;
constexpr unsigned kNormOccupancyPadBytes = 27000;   // 6 workgroups per CU
// Clip: half a piece per workgroup, two loads per lane.  604 M fp32 elements in place, norm included: 1050 us (of which the
// norm is 320; 6.6 TB/s while it reads and writes); a whole piece and four loads with 4 workgroups per CU 1060, with 3 1167,
// with 8 1103 us; one wavefront per workgroup with one load per lane 1076-1140 us.
constexpr int kScaleLoads = 2;
constexpr int kScaleParts = 2;
constexpr int kScalePartsPerXcdRun = 64;
constexpr unsigned kScaleOccupancyPadBytes = 20500;  // 7

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
template <bool KEEP>
__device__ __forceinline__ u32x4 load_grad(const char* p) { return KEEP ? ldg16(p) : ldg16_nt(p); }
template <int NORM, int D, bool KEEP>
__device__ __forceinline__ typename NormAcc<NORM>::T piece_norm(const GradPiece& p)
{
    constexpr int kVec = 16 / dtype_bytes(D), kBatch = kNormLoads * kGradThreads;
    typename NormAcc<NORM>::T a = NormAcc<NORM>::zero();
    const int t = threadIdx.x, head = head_of(p.g, dtype_bytes(D), p.n), whole = (p.n - head) / kVec;
    const char* g = p.g + head * dtype_bytes(D);
    for (int b = 0; b < whole; b += kBatch) {
        u32x4 v[kNormLoads];
        if (b + kBatch <= whole) {
#pragma unroll
            for (int i = 0; i < kNormLoads; ++i) v[i] = load_grad<KEEP>(g + (size_t)(b + i * kGradThreads + t) * 16);
        } else {  // lanes past the end load the last vector and count it as zeros
#pragma unroll
            for (int i = 0; i < kNormLoads; ++i) v[i] = load_grad<KEEP>(g + (size_t)min(b + i * kGradThreads + t, whole - 1) * 16);
#pragma unroll
            for (int i = 0; i < kNormLoads; ++i)
                if (b + i * kGradThreads + t >= whole) v[i] = (u32x4){0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < kNormLoads; ++i) add_vec<NORM, D>(a, v[i]);
    }
    if (t < head) NormAcc<NORM>::add(a, load_elem<D>(p.g, t));
    const int e = whole * kVec + t;
    if (e < p.n - head) NormAcc<NORM>::add(a, load_elem<D>(g, e));
    return a;
}

template <int NORM, bool KEEP, typename Source>
__global__ __launch_bounds__(kGradThreads) void grad_norm_partials_kernel(const Source src, const int64_t n_items, char* partials)
{
    typedef typename NormAcc<NORM>::T T;
    __shared__ T lds[kGradThreads / 64];
    const int64_t slot = (int64_t)blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
    const int64_t item = item_of_slot(slot, n_items, kNormPiecesPerXcdRun);
    GradPiece p = src.piece(item);
    asm volatile("" : "+s"(p.g), "+s"(p.n), "+s"(p.g_dtype));
    if (slot >= n_items) return;  // uniform per workgroup
    T a;
    if (p.g_dtype == WQ_DTYPE_BF16) a = piece_norm<NORM, WQ_DTYPE_BF16, KEEP>(p);
    else if (p.g_dtype == WQ_DTYPE_F16) a = piece_norm<NORM, WQ_DTYPE_F16, KEEP>(p);
    else a = piece_norm<NORM, WQ_DTYPE_F32, KEEP>(p);
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

template <int NORM, int THREADS>
__global__ __launch_bounds__(THREADS) void grad_norm_total_kernel(const char* partials, const int64_t n, const float scale,
                                                                 const float* scale_dev, float* total)
{
    typedef typename NormAcc<NORM>::T T;
    __shared__ T lds[THREADS / 64];
    const T a = fold_partials<NORM, THREADS>(partials, n, lds);
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
// A lane takes the elements of one 16-byte access of the wider of the two types; part k of a piece's workgroups takes every
// kScaleParts-th batch from batch k, the first one also what lies before the first 16-byte boundary and behind the last vector.
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
__device__ __forceinline__ void piece_scale(const GradPiece& p, int part, float c)
{
    typedef ScaleVec<G, O> Vec;
    constexpr int kBatch = kScaleLoads * kGradThreads;
    constexpr int kG = dtype_bytes(G), kO = dtype_bytes(O);
    const int t = threadIdx.x, head = kO >= kG ? head_of(p.out, kO, p.n) : head_of(p.g, kG, p.n), n = p.n - head, whole = n / Vec::kElems;
    const char* g = p.g + head * kG;
    char* out = p.out + head * kO;
    for (int b = part * kBatch; b < whole; b += kScaleParts * kBatch) {
        Vec v[kScaleLoads];
        if (b + kBatch <= whole) {
#pragma unroll
            for (int i = 0; i < kScaleLoads; ++i) v[i].load(g + (size_t)(b + i * kGradThreads + t) * Vec::kIn);
#pragma unroll
            for (int i = 0; i < kScaleLoads; ++i) v[i].scale_and_store(out + (size_t)(b + i * kGradThreads + t) * Vec::kOut, c);
        } else {  // lanes past the end load the last vector (in place perhaps as its owner stores it) and drop it
#pragma unroll
            for (int i = 0; i < kScaleLoads; ++i) v[i].load(g + (size_t)min(b + i * kGradThreads + t, whole - 1) * Vec::kIn);
#pragma unroll
            for (int i = 0; i < kScaleLoads; ++i)
                if (b + i * kGradThreads + t < whole) v[i].scale_and_store(out + (size_t)(b + i * kGradThreads + t) * Vec::kOut, c);
        }
    }
    if (part) return;
    const int e = whole * Vec::kElems + t;
    if (e < n) store_elem<O>(out, e, load_elem<G>(g, e) * c);
    if (t < head) store_elem<O>(p.out, t, load_elem<G>(p.g, t) * c);
}
template <int G>
__device__ __forceinline__ void piece_scale_from(const GradPiece& p, int part, float c)
{
    if (p.out_dtype == WQ_DTYPE_BF16) piece_scale<G, WQ_DTYPE_BF16>(p, part, c);
    else if (p.out_dtype == WQ_DTYPE_F16) piece_scale<G, WQ_DTYPE_F16>(p, part, c);
    else piece_scale<G, WQ_DTYPE_F32>(p, part, c);
}

// NORM < 0: the norm is at `total`.  Otherwise every workgroup folds the list's partials for itself - kFoldByAll at most, a
// microsecond - in the order in which the total's kernel would, and the first one writes the norm: a launch less where the
// launches are most of the time (a plan's clip of 65 pieces 11.6 -> 8.3 us, of 576 12.0 -> 9.2, of 1024 12.2 -> 11.3, of 1152
// 13.6 -> 13.5, of 2304 20.2 -> 23.1 us: every workgroup's microsecond adds up).
template <int NORM, typename Source>
__global__ __launch_bounds__(kGradThreads) void grad_scale_kernel(const Source src, const int64_t n_parts, float* total, float max_norm,
                                                                 float scale, const float* scale_dev, const Partials partials)
{
    const int64_t slot = (int64_t)blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
    const int64_t unit = item_of_slot(slot, n_parts, kScalePartsPerXcdRun);
    const int part = (int)(unit % kScaleParts);
    GradPiece p = src.piece(unit / kScaleParts);
    uint32_t norm_bits = NORM < 0 ? const_u32(total) : 0u, dev = 0u;
    if (NORM < 0) dev = const_u32(scale_dev ? scale_dev : total);
    else if (scale_dev) dev = const_u32(scale_dev);
    asm volatile("" : "+s"(p.g), "+s"(p.out), "+s"(p.n), "+s"(p.g_dtype), "+s"(p.out_dtype), "+s"(norm_bits), "+s"(dev), "+s"(max_norm), "+s"(scale));
    const float s = scale_dev ? scale * u2f(dev) : scale;
    float norm = u2f(norm_bits);
    if constexpr (NORM >= 0) {
        __shared__ typename NormAcc<NORM>::T lds[kGradThreads / 64];
        norm = NormAcc<NORM>::finish(fold_partials<NORM, kGradThreads>(partials.at, partials.n, lds), s);
        if (slot == 0 && threadIdx.x == 0) stg<float>(total, norm);
    }
    const float c = clip_coefficient(norm, max_norm, s);
    if (slot >= n_parts || (c == 1.0f && p.out == p.g)) return;  // uniform per workgroup
    if (p.g_dtype == WQ_DTYPE_BF16) piece_scale_from<WQ_DTYPE_BF16>(p, part, c);
    else if (p.g_dtype == WQ_DTYPE_F16) piece_scale_from<WQ_DTYPE_F16>(p, part, c);
    else piece_scale_from<WQ_DTYPE_F32>(p, part, c);
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

// A norm whose gradients are read again right away (`again`) leaves them in the 256 MB Infinity Cache if they fit: plain
// instead of non-temporal loads make the norm alone slower (202 MB of bf16: 35 -> 38 us) and norm and clip together faster
// (174 MB of bf16 into fp32: 119 -> 106 us, 202 MB in place 83 -> 80 us); beyond it little is left to find (fp32 in place, 336 MB
// 152.8 -> 150.4, 403 MB 181.4 -> 180.4) and then nothing (2.4 GB 1060 -> 1087 us).
// The host knows the number of pieces only: a list of more small tensors than that is taken for a long one.
constexpr int64_t kKeepPieces = (256 << 20) / WQ_GRAD_ITEM_BYTES;
// The same for an update, whose pieces are 32 KiB of fp32 or 16 KiB of bf16 gradients and which comes back to a gradient while
// it streams six arrays more; a part of a list beyond the cache is still found there.  With clip, non-temporal -> plain, fp32: 17 MB
// 30.0 -> 28.3 us, 101 MB 139 -> 129, 252 MB 342 -> 313, 403 MB 536 -> 510, 604 MB 796 -> 775, 1.2 GB 1602 -> 1592, 1.8 GB 2394 ->
// 2391, 4.8 GB 7230 -> 7279; bf16: 101 MB 242 -> 230, 252 MB 598 -> 569, 403 MB 949 -> 921, 0.8 GB 1907 -> 1890, 1.2 GB 2860 -> 2852,
// 1.8 GB 4298 -> 4315.  32768 pieces are 1.1 GB of fp32 or 0.5 GB of bf16.
constexpr int64_t kKeepAdamItems = 32768;

template <int NORM, typename Source>
static void launch_pieces(const Source& src, int64_t n_items, bool keep, char* partials, hipStream_t st)
{
    if (n_items == 0) return;
    const dim3 g = grid_for_items(n_items);
    if (keep) grad_norm_partials_kernel<NORM, true><<<g, kGradThreads, kNormOccupancyPadBytes, st>>>(src, n_items, partials);
    else grad_norm_partials_kernel<NORM, false><<<g, kGradThreads, kNormOccupancyPadBytes, st>>>(src, n_items, partials);
}
template <int NORM>
static Partials launch_fold(char* partials, int64_t n_items, hipStream_t st)
{
    if (n_items <= kFoldDirect) return {partials, n_items};
    const int64_t groups = cdiv64(n_items, kFoldGroup);
    char* sums = partials + n_items * 8;
    grad_norm_fold_kernel<NORM><<<(unsigned)groups, kGradThreads, 0, st>>>(partials, n_items, sums);
    return {sums, groups};
}
constexpr int64_t kFoldByAll = 1024;
template <int NORM>
static void launch_total(char* partials, int64_t n_items, float scale, const float* scale_dev, float* total, hipStream_t st)
{
    const Partials p = launch_fold<NORM>(partials, n_items, st);
    if (n_items <= kFoldByAll) grad_norm_total_kernel<NORM, kGradThreads><<<1, kGradThreads, 0, st>>>(p.at, p.n, scale, scale_dev, total);
    else grad_norm_total_kernel<NORM, 1024><<<1, 1024, 0, st>>>(p.at, p.n, scale, scale_dev, total);
}
template <int NORM>
static Partials launch_update_partials(const TableSource& src, int64_t n_items, void* workspace, hipStream_t st)
{
    launch_pieces<NORM>(src, n_items, n_items <= kKeepAdamItems, partials_of(workspace), st);
    return launch_fold<NORM>(partials_of(workspace), n_items, st);
}
Partials launch_norm_partials(const TableSource& src, int64_t n_items, int norm, void* workspace, hipStream_t st)
{
    return norm == WQ_NORM_2 ? launch_update_partials<WQ_NORM_2>(src, n_items, workspace, st)
                             : launch_update_partials<WQ_NORM_INF>(src, n_items, workspace, st);
}
template <int NORM>
static void launch_table_norm(const TableSource& src, int64_t n_items, bool again, float scale, const float* scale_dev, void* workspace,
                              float* total, hipStream_t st)
{
    launch_pieces<NORM>(src, n_items, again && n_items <= kKeepPieces, partials_of(workspace), st);
    launch_total<NORM>(partials_of(workspace), n_items, scale, scale_dev, total, st);
}
template <int NORM, typename Source>
static void launch_scale(const Source& src, int64_t n_items, float* total, float max_norm, float scale, const float* scale_dev,
                         Partials partials, hipStream_t st)
{
    if (n_items == 0) return;
    const int64_t parts = n_items * kScaleParts;
    grad_scale_kernel<NORM><<<grid_for_items(parts), kGradThreads, kScaleOccupancyPadBytes, st>>>(src, parts, total, max_norm, scale,
                                                                                                   scale_dev, partials);
}
template <int NORM>
static void launch_table_clip(const TableSource& src, int64_t n_items, float max_norm, float scale, const float* scale_dev,
                              void* workspace, float* total, hipStream_t st)
{
    if (n_items == 0 || n_items > kFoldByAll) {
        launch_table_norm<NORM>(src, n_items, true, scale, scale_dev, workspace, total, st);
        launch_scale<-1>(src, n_items, total, max_norm, scale, scale_dev, Partials{}, st);
    } else {
        launch_pieces<NORM>(src, n_items, true, partials_of(workspace), st);
        launch_scale<NORM>(src, n_items, total, max_norm, scale, scale_dev, Partials{partials_of(workspace), n_items}, st);
    }
}

static bool grad_dtype_ok(int d) { return d == WQ_DTYPE_BF16 || d == WQ_DTYPE_F16 || d == WQ_DTYPE_F32; }

// ---- HOST lists -----------------------------------------------------------------------------------------------------------
struct HostList {
    const void* const* g;
    const int64_t* n;
    const int32_t* dtype;
    int n_tensors;
    int64_t pieces(int i) const { return pieces_of(n[i], grad_item(dtype[i]), phase_of(g[i], dtype_bytes(dtype[i]))); }
};
// number of pieces of the whole list; negative: an error.  Looks at everything before anything is launched.
static int64_t check_list(const HostList& l)
{
    if (l.n_tensors < 0) return WQ_ERR_SHAPE;
    if (l.n_tensors && (!l.g || !l.n || !l.dtype)) return WQ_ERR_NULL;
    int64_t total = 0;
    for (int i = 0; i < l.n_tensors; ++i) {
        if (l.n[i] < 0) return WQ_ERR_SHAPE;
        if (!grad_dtype_ok(l.dtype[i])) return WQ_ERR_MODE;
        if (l.n[i] > ((int64_t)1 << 40)) return WQ_ERR_TOO_LARGE;
        if (l.n[i] && !l.g[i]) return WQ_ERR_NULL;
        if ((uintptr_t)l.g[i] % dtype_bytes(l.dtype[i])) return WQ_ERR_ALIGN;
        total += l.pieces(i);
        if (total > ((int64_t)1 << 31) - 1) return WQ_ERR_TOO_LARGE;
    }
    return total;
}
// calls launch(source, pieces of it, pieces before it) for every WQ_GRAD_LIST_LAUNCH tensors that have elements
template <typename Launch>
static void for_each_launch(const HostList& l, Launch launch)
{
    ListSource src;
    int k = 0;
    int64_t items = 0, before = 0;
    for (int i = 0; i < l.n_tensors; ++i) {
        if (l.n[i] == 0) continue;
        src.g[k] = (const char*)l.g[i];
        src.n_dtype[k] = (uint64_t)l.n[i] | (uint64_t)l.dtype[i] << 56;
        src.start[k++] = (int32_t)items;
        items += l.pieces(i);
        if (k == WQ_GRAD_LIST_LAUNCH) {
            src.n_tensors = k;
            launch(src, items, before);
            before += items;
            k = 0, items = 0;
        }
    }
    src.n_tensors = k;
    if (k) launch(src, items, before);
}
template <int NORM>
static void launch_list_pieces(const HostList& l, bool keep, char* partials, hipStream_t st)
{
    for_each_launch(l, [&](const ListSource& src, int64_t items, int64_t before) { launch_pieces<NORM>(src, items, keep, partials + before * 8, st); });
}
template <int NORM>
static void launch_list_norm(const HostList& l, int64_t pieces, float scale, void* workspace, float* total, hipStream_t st)
{
    launch_list_pieces<NORM>(l, false, partials_of(workspace), st);
    launch_total<NORM>(partials_of(workspace), pieces, scale, nullptr, total, st);
}
static void launch_list_scale(const HostList& l, float* total, float max_norm, float scale, hipStream_t st)
{
    for_each_launch(l, [&](const ListSource& src, int64_t items, int64_t) { launch_scale<-1>(src, items, total, max_norm, scale, nullptr, Partials{}, st); });
}
template <int NORM>
static void launch_list_clip(const HostList& l, int64_t pieces, float max_norm, float scale, void* workspace, float* total, hipStream_t st)
{
    char* partials = partials_of(workspace);
    launch_list_pieces<NORM>(l, pieces <= kKeepPieces, partials, st);
    if (pieces == 0 || pieces > kFoldByAll || l.n_tensors > WQ_GRAD_LIST_LAUNCH) {
        launch_total<NORM>(partials, pieces, scale, nullptr, total, st);
        launch_list_scale(l, total, max_norm, scale, st);
    } else {
        for_each_launch(l, [&](const ListSource& src, int64_t items, int64_t) {
            launch_scale<NORM>(src, items, total, max_norm, scale, nullptr, Partials{partials, pieces}, st);
        });
    }
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
    const TableSource src = {(const int64_t*)items, words};
    if (norm == WQ_NORM_2) launch_table_norm<WQ_NORM_2>(src, n_items, false, grad_scale, grad_scale_dev, workspace, total, st);
    else launch_table_norm<WQ_NORM_INF>(src, n_items, false, grad_scale, grad_scale_dev, workspace, total, st);
    if (each && n_desc) {
        const char* partials = partials_of(workspace);
        if (norm == WQ_NORM_2) grad_norm_each_kernel<WQ_NORM_2><<<n_desc, kGradThreads, 0, st>>>(partials, item_start, grad_scale, grad_scale_dev, each);
        else grad_norm_each_kernel<WQ_NORM_INF><<<n_desc, kGradThreads, 0, st>>>(partials, item_start, grad_scale, grad_scale_dev, each);
    }
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}

WQ_EXPORT int64_t wq_grad_list_workspace_bytes(const void* const* g, const int64_t* n, const int32_t* dtype, int n_tensors)
{
    const int64_t pieces = check_list({g, n, dtype, n_tensors});
    return pieces < 0 ? 0 : wq_grad_workspace_bytes(pieces);
}

WQ_EXPORT int wq_grad_norm_list(const void* const* g, const int64_t* n, const int32_t* dtype, int n_tensors, int norm, float grad_scale,
                                void* workspace, float* total, void* stream)
{
    if (norm != WQ_NORM_2 && norm != WQ_NORM_INF) return WQ_ERR_MODE;
    const HostList l = {g, n, dtype, n_tensors};
    const int64_t pieces = check_list(l);
    if (pieces < 0) return (int)pieces;
    if (!workspace || !total) return WQ_ERR_NULL;
    if (norm == WQ_NORM_2) launch_list_norm<WQ_NORM_2>(l, pieces, grad_scale, workspace, total, (hipStream_t)stream);
    else launch_list_norm<WQ_NORM_INF>(l, pieces, grad_scale, workspace, total, (hipStream_t)stream);
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
    hipStream_t st = (hipStream_t)stream;
    const TableSource src = {(const int64_t*)items, 4};
    if (total_given) launch_scale<-1>(src, n_items, const_cast<float*>(total_given), max_norm, grad_scale, grad_scale_dev, Partials{}, st);
    else if (norm == WQ_NORM_2) launch_table_clip<WQ_NORM_2>(src, n_items, max_norm, grad_scale, grad_scale_dev, workspace, total, st);
    else launch_table_clip<WQ_NORM_INF>(src, n_items, max_norm, grad_scale, grad_scale_dev, workspace, total, st);
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}

WQ_EXPORT int wq_grad_clip_list(void* const* g, const int64_t* n, const int32_t* dtype, int n_tensors, int norm, float max_norm,
                                float grad_scale, const float* total_given, void* workspace, float* total, void* stream)
{
    if (norm != WQ_NORM_2 && norm != WQ_NORM_INF) return WQ_ERR_MODE;
    const HostList l = {g, n, dtype, n_tensors};
    const int64_t pieces = check_list(l);
    if (pieces < 0) return (int)pieces;
    if (!total_given && (!workspace || !total)) return WQ_ERR_NULL;
    if (pieces == 0 && total_given) return WQ_OK;
    hipStream_t st = (hipStream_t)stream;
    if (total_given) launch_list_scale(l, const_cast<float*>(total_given), max_norm, grad_scale, st);
    else if (norm == WQ_NORM_2) launch_list_clip<WQ_NORM_2>(l, pieces, max_norm, grad_scale, workspace, total, st);
    else launch_list_clip<WQ_NORM_INF>(l, pieces, max_norm, grad_scale, workspace, total, st);
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}
