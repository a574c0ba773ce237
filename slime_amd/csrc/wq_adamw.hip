// One AdamW step over many tensors for gfx950: fp32 weights and moments, gradients in bf16, fp16 or fp32, the clip folded
// in, and the bf16 / fp16 copy of the new weight - what a weight sync quantises - written by the same pass.
//
//   t = step + 1, g' = c g, p1 = p (1 - lr l w), m = b1 m + (1 - b1) g', v = b2 v + (1 - b2) g'^2
//   p = p1 - lr l / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps), out = round(p)
//
// Bound by HBM: 24 bytes of state and 2 or 4 of gradient per element, plus 2 for the copy.  The step number lives on the
// device and one workgroup works out the step's scalars (bias corrections in 64 bits), so a recorded step replays with
// the right ones.

#include "wq_grad_common.h"

#include <math.h>

namespace wq {

// One wavefront per workgroup and one 16-byte access per lane and stream (256 elements), 12 of them on a CU by an unused
// dynamic LDS allocation: eight streams at once want few bytes in flight and short-lived workgroups.  604 M elements with
// fp32 gradients, norm (330 us) included: 3150-3190 us, 6.4 TB/s in the update, where the best of 1800 shapes of a bare kernel
// without any table got 6.43; 256 threads on 2048 elements and 3 workgroups per CU 3290, on 1024 and 4 3380, on 2048 and 8
// 3600 us; `nt` instead of `nt sc1` stores 3250 us; 15 wavefronts on a CU 3300 us.  Runs of 512 parts per XCD rather than 256: the
// same at this size, 326 for 334 us on 75 M elements.  807 M elements with bf16 gradients: 3770 us (219 of norm).
constexpr int kAdamThreads = 64;
constexpr int kAdamPart = 256;                        // elements of a workgroup
constexpr int kAdamParts = kAdamItem / kAdamPart;
constexpr int kAdamPartsPerXcdRun = 512;
constexpr unsigned kAdamOccupancyPadBytes = 13000;

struct AdamControl {       // at the start of the workspace, written anew by every step
    float coefficient;
    float lr;
    float step_size;       // lr / (1 - b1^t)
    float inv_sqrt_bc2;    // 1 / sqrt(1 - b2^t)
    int32_t skip;
    int32_t unused[3];
};
typedef uint32_t u32x8 __attribute__((ext_vector_type(8), aligned(16)));     // a workspace has no more
static_assert(sizeof(AdamControl) == sizeof(u32x8) && sizeof(AdamControl) <= kGradControlBytes, "workspace layout");

struct AdamBeginArgs {
    const char* partials;
    int64_t n_partials;
    double log_beta1, log_beta2, lr;     // -inf for a beta of 0
    const float* lr_dev;
    const float* grad_scale_dev;
    const float* total_given;
    float* total;
    int64_t* step;
    float grad_scale, max_norm;
    int32_t need_norm, skip_nonfinite;
};

template <int NORM>
__global__ __launch_bounds__(1024) void adamw_begin_kernel(const AdamBeginArgs a, AdamControl* control)
{
    typedef typename NormAcc<NORM>::T T;
    __shared__ T lds[16];
    __shared__ double corrections[2];
    const float scale = effective_scale(a.grad_scale, a.grad_scale_dev);
    const int64_t t = ldg<int64_t>(a.step) + 1;
    // 1 - beta^t = -expm1(t ln beta), each by a wavefront of its own while the others' partials are on their way
    if (threadIdx.x == 64) corrections[0] = -expm1((double)t * a.log_beta1);
    if (threadIdx.x == 128) corrections[1] = -expm1((double)t * a.log_beta2);
    float norm = 0.0f;
    if (a.need_norm && a.total_given) norm = ldg<float>(a.total_given);
    else if (a.need_norm) norm = NormAcc<NORM>::finish(fold_partials<NORM, 1024>(a.partials, a.n_partials, lds), scale);
    __syncthreads();
    if (threadIdx.x) return;
    if (a.need_norm && !a.total_given) stg<float>(a.total, norm);
    const bool skip = a.skip_nonfinite && !(norm <= 3.4028234663852886e38f);
    const double lr = a.lr_dev ? a.lr * (double)ldg<float>(a.lr_dev) : a.lr;
    WQ_GLOBAL AdamControl* out = (WQ_GLOBAL AdamControl*)control;
    out->coefficient = a.max_norm >= 0.0f ? clip_coefficient(norm, a.max_norm, scale) : scale;
    out->lr = (float)lr;
    out->step_size = (float)(lr / corrections[0]);
    out->inv_sqrt_bc2 = (float)(1.0 / sqrt(corrections[1]));
    out->skip = skip;
    if (!skip) stg<int64_t>(a.step, t);
}

struct AdamConsts {
    float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
};
struct AdamStep {          // the constants of a piece
    float c, decay, step_size, inv_sqrt_bc2;
};

__device__ __forceinline__ void adam_elem(float g, float& p, float& m, float& v, const AdamConsts& k, const AdamStep& s)
{
    g *= s.c;
    m = __builtin_fmaf(k.one_minus_beta1, g, k.beta1 * m);
    v = __builtin_fmaf(k.one_minus_beta2 * g, g, k.beta2 * v);
    const float denom = __builtin_fmaf(__builtin_sqrtf(v), s.inv_sqrt_bc2, k.eps);
    p = __builtin_fmaf(-s.step_size, m / denom, __builtin_fmaf(-s.decay, p, p));
}

struct AdamPart {
    const char* g;
    char *p, *m, *v, *o;
    int n, g_dtype, out_dtype;
};

template <int G, int O>     // O < 0: no copy
__device__ __forceinline__ void adam_part(const AdamPart& d, const AdamConsts& k, const AdamStep& s)
{
    const int head = head_of(d.p, 4, d.n), whole = (d.n - head) / 4;
    const char* g = d.g + head * dtype_bytes(G);
    char *p = d.p + head * 4, *m = d.m + head * 4, *v = d.v + head * 4, *o = d.o + head * 2;
    for (int i = threadIdx.x; i < whole; i += kAdamThreads) {
        const uint32_t at = (uint32_t)i * 16u;
        float gf[4];
        if constexpr (G == WQ_DTYPE_F32) {
            const u32x4 w = ldg16_nt(g + at);
            gf[0] = u2f(w.x), gf[1] = u2f(w.y), gf[2] = u2f(w.z), gf[3] = u2f(w.w);
        } else {
            const u32x2 w = ldg8_nt(g + at / 2);
            const f32x2 a = unpack2<G>(w.x), b = unpack2<G>(w.y);
            gf[0] = a.x, gf[1] = a.y, gf[2] = b.x, gf[3] = b.y;
        }
        u32x4 pw = ldg16_nt(p + at), mw = ldg16_nt(m + at), vw = ldg16_nt(v + at);
        float pf[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float mf = u2f(mw[e]), vf = u2f(vw[e]);
            pf[e] = u2f(pw[e]);
            adam_elem(gf[e], pf[e], mf, vf, k, s);
            pw[e] = f2u(pf[e]), mw[e] = f2u(mf), vw[e] = f2u(vf);
        }
        stg_nt_sc1<u32x4>(p + at, pw);
        stg_nt_sc1<u32x4>(m + at, mw);
        stg_nt_sc1<u32x4>(v + at, vw);
        if constexpr (O >= 0) stg_nt_sc1<u32x2>(o + at / 2, (u32x2){pack2<O>(pf[0], pf[1]), pack2<O>(pf[2], pf[3])});
    }
    // before the first boundary and behind the last vector: a lane per element
    const int t = threadIdx.x, behind = head + whole * 4;
    const int e = t < head ? t : behind + t - head;
    if (e < d.n) {
        float pf = ldg<float>(d.p + (size_t)e * 4), mf = ldg<float>(d.m + (size_t)e * 4), vf = ldg<float>(d.v + (size_t)e * 4);
        adam_elem(load_elem<G>(d.g, e), pf, mf, vf, k, s);
        stg<float>(d.p + (size_t)e * 4, pf);
        stg<float>(d.m + (size_t)e * 4, mf);
        stg<float>(d.v + (size_t)e * 4, vf);
        if constexpr (O >= 0) store_elem<O>(d.o, e, pf);
    }
}
template <int G>
__device__ __forceinline__ void adam_part_from(const AdamPart& d, const AdamConsts& k, const AdamStep& s)
{
    if (!d.o) adam_part<G, -1>(d, k, s);
    else if (d.out_dtype == WQ_DTYPE_BF16) adam_part<G, WQ_DTYPE_BF16>(d, k, s);
    else adam_part<G, WQ_DTYPE_F16>(d, k, s);
}

__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(const wq_adamw_desc* items, const int64_t n_parts, AdamConsts k,
                                                            const AdamControl* control)
{
    const int64_t slot = (int64_t)blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
    const int64_t part = item_of_slot(slot, n_parts, kAdamPartsPerXcdRun);
    i64x8 w = *(const WQ_CONST i64x8*)((const int64_t*)items + part / kAdamParts * 8);
    u32x8 cw = *(const WQ_CONST u32x8*)control;
    asm volatile("" : "+s"(w), "+s"(cw), "+s"(k.beta1), "+s"(k.one_minus_beta1), "+s"(k.beta2), "+s"(k.one_minus_beta2), "+s"(k.eps));
    const AdamControl c = __builtin_bit_cast(AdamControl, cw);
    if (slot >= n_parts || c.skip) return;  // uniform per workgroup
    const wq_adamw_desc d = __builtin_bit_cast(wq_adamw_desc, w);
    const Run r = run_of(part % kAdamParts, d.n, kAdamPart, phase_of(d.p, 4));
    if (r.n <= 0) return;
    const int at = (int)r.at;
    const AdamPart a = {(const char*)d.g + at * dtype_bytes(d.g_dtype), (char*)(d.p + at), (char*)(d.m + at), (char*)(d.v + at),
                        d.out ? (char*)d.out + at * 2 : nullptr, r.n, d.g_dtype, d.out_dtype};
    const AdamStep s = {c.coefficient, c.lr * d.lr_scale * d.weight_decay, c.step_size * d.lr_scale, c.inv_sqrt_bc2};
    if (a.g_dtype == WQ_DTYPE_BF16) adam_part_from<WQ_DTYPE_BF16>(a, k, s);
    else if (a.g_dtype == WQ_DTYPE_F16) adam_part_from<WQ_DTYPE_F16>(a, k, s);
    else adam_part_from<WQ_DTYPE_F32>(a, k, s);
}

}  // namespace wq

using namespace wq;

WQ_EXPORT int wq_adamw_items(const wq_adamw_desc* items, int64_t n_items, const wq_adamw_hyper* h, void* workspace, void* stream)
{
    if (n_items < 0) return WQ_ERR_SHAPE;
    if (!h || !workspace || !h->step || (n_items && !items)) return WQ_ERR_NULL;
    if (h->norm != WQ_NORM_2 && h->norm != WQ_NORM_INF) return WQ_ERR_MODE;
    if (!(h->beta1 >= 0.0 && h->beta1 < 1.0 && h->beta2 >= 0.0 && h->beta2 < 1.0 && h->eps >= 0.0)) return WQ_ERR_SHAPE;
    if (h->eps > 0.0 && (float)h->eps == 0.0f) return WQ_ERR_SHAPE;   // 0 / 0 where the formula has 0
    const bool need_norm = h->max_norm >= 0.0f || h->skip_nonfinite;
    if (need_norm && !h->total_given && !h->total) return WQ_ERR_NULL;
    hipStream_t st = (hipStream_t)stream;
    AdamBeginArgs a = {};
    a.log_beta1 = log(h->beta1);
    a.log_beta2 = log(h->beta2);
    a.lr = h->lr;
    a.lr_dev = h->lr_dev;
    a.grad_scale_dev = h->grad_scale_dev;
    a.total_given = h->total_given;
    a.total = h->total;
    a.step = h->step;
    a.grad_scale = h->grad_scale;
    a.max_norm = h->max_norm;
    a.need_norm = need_norm;
    a.skip_nonfinite = h->skip_nonfinite;
    if (need_norm && !h->total_given) {
        const Partials p = launch_norm_partials(TableSource{(const int64_t*)items, 8}, n_items, h->norm, workspace, st);
        a.partials = p.at;
        a.n_partials = p.n;
    }
    AdamControl* control = (AdamControl*)workspace;
    if (h->norm == WQ_NORM_2) adamw_begin_kernel<WQ_NORM_2><<<1, 1024, 0, st>>>(a, control);
    else adamw_begin_kernel<WQ_NORM_INF><<<1, 1024, 0, st>>>(a, control);
    if (n_items) {
        const AdamConsts k = {(float)h->beta1, (float)(1.0 - h->beta1), (float)h->beta2, (float)(1.0 - h->beta2), (float)h->eps};
        const int64_t parts = n_items * kAdamParts;
        adamw_kernel<<<grid_for_items(parts), kAdamThreads, kAdamOccupancyPadBytes, st>>>(items, parts, k, control);
    }
    WQ_LAUNCH_CHECK();
    return WQ_OK;
}
