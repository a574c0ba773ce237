"""Gradient norm, clip and AdamW update against the definitions in 64 bits.

Tolerances count roundings (u = 2^-24, half a step of fp32; h = half a step of the output type):
- a 2-norm is summed in 64 bits and rounded once: u (n * 2^-53 is far below it); an infinity norm is exact; a scale other than
  one is another rounding in the infinity norm;
- a coefficient takes the norm (u), + 1e-6f (u, and u for the constant), the division (u), the scale (u): 5 u; the product with
  the gradient one more: 6 u; the output h, or half its smallest subnormal;
- the update's are written at ``adamw_bounds``.
"""

import math

import pytest
import torch

import slime_amd
from slime_amd import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SUBNORMAL = {BF16: 2.0 ** -133, F16: 2.0 ** -24, F32: 2.0 ** -149}
ITEM = 16384
# one element; empty; around one piece and its 256-lane rows; several pieces; odd matrices
SIZES = [(1,), (0,), (), (ITEM,), (ITEM - 1,), (ITEM + 1,), (2047,), (2049,), (3 * ITEM + 5,), (7, 7168), (129, 257), (300, 520)]


def tensors(shapes, dtypes, seed=0, scale=1.0, offset=0, device="cuda:0"):
    """Random tensors of the shapes, each ``offset`` elements into an allocation of its own, guards behind it."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        d = dtypes[i % len(dtypes)]
        n = math.prod(s)
        buf = torch.full((n + offset + 64,), 7.0, dtype=d, device=device)
        t = buf[offset:offset + n]
        t.copy_((torch.randn(n, generator=g) * scale).to(d))
        t = t.view(s)
        t.guard = (buf, offset, n)
        out.append(t)
    return out


def check_guards(ts):
    for t in ts:
        buf, offset, n = t.guard
        assert bool((buf[:offset] == 7).all()) and bool((buf[offset + n:] == 7).all())


def norm_of(ts, norm_type=2.0):
    xs = [t.double().reshape(-1) for t in ts if t.numel()]
    if not xs:
        return 0.0
    if norm_type == math.inf:
        return max(x.abs().max().item() for x in xs)
    return math.sqrt(sum(x.square().sum().item() for x in xs))


def check_norm(got, ts, norm_type=2.0, scale=1.0):
    want = norm_of(ts, norm_type) * scale
    assert got.dtype == F32 and got.dim() == 0
    assert abs(got.item() - want) <= 1.001 * U * want * (1 if norm_type == 2.0 or scale == 1.0 else 2) + 2.0 ** -150, (got.item(), want)


# ---- norm -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [[BF16], [F16], [F32], [F32, BF16, F16]])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_norm_function_and_plan(cuda, norm_type, dtypes, offset):
    ts = tensors(SIZES, dtypes, 1, 0.3, offset)
    check_norm(slime_amd.get_total_norm(ts, norm_type), ts, norm_type)
    check_norm(slime_amd.get_total_norm(ts[8], norm_type), ts[8:9], norm_type)
    plan = slime_amd.GradNormPlan(ts, norm_type, per_tensor=True)
    total, each = plan.run()
    check_norm(total, ts, norm_type)
    assert each.shape == (len(ts),)
    for e, t in zip(each, ts):
        check_norm(e, [t], norm_type)
    first = total.clone(), each.clone()
    for t in ts:
        t.mul_(0.5)
    total, each = plan.run(grad_scale=2.0)                 # exact factors of two: the same bits
    assert torch.equal(total, first[0]) and torch.equal(each, first[1])
    scale = torch.tensor(0.37, device=cuda)
    check_norm(plan.run(grad_scale=scale)[0], ts, norm_type, scale.item())


@pytest.mark.parametrize("n", [1, 175, 176, 177, 400])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_norm_over_many_tensors(cuda, n, norm_type):
    """176 tensors travel in the arguments of one launch."""
    ts = tensors([(1 + 37 * i % 5000,) for i in range(n)], [BF16, F32], 2, 0.1)
    check_norm(slime_amd.get_total_norm(ts, norm_type), ts, norm_type)
    check_norm(slime_amd.get_total_norm((t for t in ts), norm_type), ts, norm_type)
    assert torch.equal(slime_amd.get_total_norm(ts, norm_type), slime_amd.GradNormPlan(ts, norm_type).run())


@pytest.mark.parametrize("dtype,value", [(F32, 1e30), (F32, 1e-30), (F32, 1e-44), (BF16, 1e30), (BF16, 1e-38), (F16, 60000.0), (F16, 2.0 ** -24)])
def test_norm_neither_overflows_nor_vanishes(cuda, dtype, value):
    t = torch.full((ITEM + 77,), value, dtype=dtype, device=cuda)
    check_norm(slime_amd.get_total_norm([t]), [t])
    check_norm(slime_amd.get_total_norm([t], math.inf), [t], math.inf)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_norm_of_nonfinite(cuda, dtype, norm_type):
    for bad, at in ((math.inf, 0), (-math.inf, ITEM + 3), (math.nan, 2 * ITEM + 8), (math.nan, 5)):
        ts = tensors([(100,), (2 * ITEM + 9,)], [dtype], 3)
        ts[1][at] = bad
        for total in (slime_amd.get_total_norm(ts, norm_type), slime_amd.GradNormPlan(ts, norm_type).run()):
            assert math.isnan(total.item()) if math.isnan(bad) else total.item() == math.inf
        with pytest.raises(RuntimeError, match="non-finite"):
            slime_amd.get_total_norm(ts, norm_type, error_if_nonfinite=True)
    ts[0][0], ts[1][5] = math.inf, math.nan              # NaN wins over infinity
    assert math.isnan(slime_amd.get_total_norm(ts, norm_type).item())


def test_norm_of_nothing(cuda):
    ts = tensors([(0,), (0, 5)], [F32])
    assert slime_amd.get_total_norm(ts).item() == 0.0
    total, each = slime_amd.GradNormPlan(ts, per_tensor=True).run()
    assert total.item() == 0.0 and each.tolist() == [0.0, 0.0]
    z = tensors([(0,), (5,), (0,), (0,), (9,)], [F32], 4)
    total, each = slime_amd.GradNormPlan(z, per_tensor=True).run()
    check_norm(total, z)
    assert each[0].item() == each[2].item() == each[3].item() == 0.0


def test_norm_takes_any_strides(cuda):
    x = tensors([(40, 30, 20)], [F32], 5)[0]
    views = [x.permute(2, 0, 1), x[:, :7], x[..., ::3], x[1:2, :1].expand(4, 5, 20), x[3].t()]
    for v in views:
        check_norm(slime_amd.get_total_norm([v]), [v])
    check_norm(slime_amd.get_total_norm([x, x]), [x, x])   # twice in the list counts twice
    check_norm(slime_amd.GradNormPlan([x, x.permute(1, 2, 0)]).run(), [x, x])


def test_norm_is_reproducible(cuda):
    ts = tensors([(513, 1027)] * 40, [BF16], 6)
    plan = slime_amd.GradNormPlan(ts, per_tensor=True)
    first = [x.clone() for x in plan.run()]
    for _ in range(5):
        again = plan.run()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---- clip -----------------------------------------------------------------------------------------------------------------
def check_clip(out, grads, max_norm, norm, scale=1.0):
    """``out`` against the definition on (64-bit copies of) ``grads``; norm: that of the scaled gradients."""
    c = scale * min(1.0, max_norm / (norm + 1e-6))
    for o, g in zip(out, grads):
        want = g.double() * c
        half = 0.0 if o.dtype == F32 else torch.finfo(o.dtype).eps / 2
        err = (o.double() - want).abs()
        assert bool((err <= want.abs() * (6 * U + half * 1.001) + SUBNORMAL[o.dtype] / 2 + SUBNORMAL[F32]).all()), (o.dtype, o.shape)


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [[BF16], [F16], [F32], [F32, BF16, F16]])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_clip_in_place(cuda, norm_type, dtypes, offset):
    for many in (False, True):
        ts = tensors(SIZES * (16 if many else 1), dtypes, 7, 0.2, offset)
        before = [t.double() for t in ts]
        max_norm = 0.31 * norm_of(ts, norm_type)
        if many:
            ps = [torch.nn.Parameter(torch.empty_like(t)) for t in ts] + [torch.nn.Parameter(torch.zeros(2, device=cuda))]
            for p, t in zip(ps, ts):
                p.grad = t
            total = slime_amd.clip_grad_norm_(ps, max_norm, norm_type)
        else:
            total = slime_amd.GradClipPlan(ts, norm_type).run(max_norm)
        check_norm(total, before, norm_type)
        check_clip(ts, before, max_norm, norm_of(before, norm_type))
        check_guards(ts)


@pytest.mark.parametrize("g_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("o_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("g_off,o_off", [(0, 0), (1, 0), (0, 3), (5, 2)])
def test_clip_into_other_tensors(cuda, g_dtype, o_dtype, g_off, o_off):
    ts, out = tensors(SIZES, [g_dtype], 8, 0.2, g_off), tensors(SIZES, [o_dtype], 9, 1.0, o_off)
    before = [t.clone() for t in ts]
    plan = slime_amd.GradClipPlan(ts, out=out)
    for max_norm, scale in ((0.5 * norm_of(ts), 1.0), (1e9, 1.0), (0.5 * norm_of(ts), 1.0 / 64), (0.004 * norm_of(ts), 1.0 / 64)):
        for o in out:
            o.fill_(3)
        total = plan.run(max_norm, grad_scale=scale)
        check_norm(total, before, scale=scale)
        check_clip(out, before, max_norm, norm_of(before) * scale, scale)
        assert all(torch.equal(a, b) for a, b in zip(ts, before))
    check_guards(ts + out)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_clip_leaves_small_gradients_alone(cuda, dtype):
    ts = tensors(SIZES, [dtype], 10, 0.1)
    before = [t.clone() for t in ts]
    plan = slime_amd.GradClipPlan(ts)
    plan.run(2.0 * norm_of(ts))
    plan.run(math.inf)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    plan.run(2.0 * norm_of(ts), grad_scale=0.5)            # the scale alone
    assert all(torch.equal(a, b * 0.5) for a, b in zip(ts, before))


def test_clip_to_nothing_and_signs_of_zero(cuda):
    for dtype in (BF16, F16, F32):
        t = torch.tensor([0.0, -0.0, 1.0, -1.0] * 9, dtype=dtype, device=cuda)
        slime_amd.GradClipPlan([t]).run(0.0)
        assert t.eq(0).all() and torch.equal(torch.signbit(t), torch.tensor([False, True] * 18, device=cuda))
        z = torch.zeros(5, dtype=dtype, device=cuda)
        assert slime_amd.GradClipPlan([z]).run(1.0).item() == 0.0 and z.eq(0).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_clip_with_nonfinite_norms(cuda, dtype):
    """As torch has it: an infinite norm clips to zero (infinities to NaN), a NaN norm makes everything NaN."""
    t = torch.randn(100, device=cuda).to(dtype)
    t[3] = math.inf
    p = torch.nn.Parameter(torch.zeros_like(t))
    p.grad = t.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        slime_amd.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert torch.equal(p.grad, t)
    assert slime_amd.clip_grad_norm_(p, 1.0).item() == math.inf
    assert math.isnan(p.grad[3].item()) and p.grad.isnan().sum().item() == 1 and p.grad.nan_to_num().eq(0).all()
    p.grad = t.clone().fill_(1.0)
    p.grad[7] = math.nan
    assert math.isnan(slime_amd.clip_grad_norm_(p, 1.0).item()) and p.grad.isnan().all()


def test_clip_by_a_given_norm(cuda):
    ts = tensors(SIZES, [BF16, F32], 11, 0.2)
    before = [t.clone() for t in ts]
    ps = [torch.nn.Parameter(torch.empty_like(t)) for t in ts]
    for p, t in zip(ps, ts):
        p.grad = t
    for norm in (torch.tensor(50.0, device=cuda), torch.tensor([50.0], dtype=torch.float64), torch.tensor(50.0, dtype=BF16, device=cuda)):
        for t, b in zip(ts, before):
            t.copy_(b)
        assert slime_amd.clip_grads_with_norm_(ps, 2.0, norm) is None
        check_clip(ts, before, 2.0, 50.0)
    for t, b in zip(ts, before):
        t.copy_(b)
    norm = torch.tensor(50.0, device=cuda)
    assert slime_amd.GradClipPlan(ts).run(2.0, total_norm=norm) is norm
    check_clip(ts, before, 2.0, 50.0)
    with pytest.raises(ValueError, match="total_norm"):
        slime_amd.GradClipPlan(ts).run(2.0, total_norm=norm.double())


def test_clip_takes_any_strides_and_refuses_shared_memory(cuda):
    x = tensors([(40, 30, 20)], [F32], 12)[0]
    before = x.clone()
    p = [torch.nn.Parameter(torch.zeros(s, device=cuda)) for s in ((40, 7, 20), (20, 40, 13), (40, 10, 10))]
    p[0].grad, p[1].grad, p[2].grad = x[:, :7], x[:, 7:20].permute(2, 0, 1), x[:, 20:, ::2]
    parts = [q.grad.double() for q in p]
    check_norm(slime_amd.clip_grad_norm_(p, 5.0), parts)
    check_clip([q.grad for q in p], parts, 5.0, norm_of(parts))
    assert torch.equal(x[:, 20:, 1::2], before[:, 20:, 1::2])          # what lies between stays
    p[1].grad = x.new_zeros(1).expand(20, 40, 13)
    with pytest.raises(ValueError, match="share memory"):
        slime_amd.clip_grad_norm_(p[:2], 5.0)
    p[0].grad = torch.ones(40, 7, 20, device=cuda)
    q = torch.nn.Parameter(torch.zeros(40, 7, 20, device=cuda))
    q.grad = p[0].grad
    with pytest.raises(ValueError, match="share memory"):
        slime_amd.clip_grad_norm_([p[0], q], 5.0)
    with pytest.raises(ValueError, match="share memory"):
        slime_amd.clip_grad_norm_([p[0], p[0]], 5.0)


@pytest.mark.parametrize("n", [3, 200])
def test_functions_keep_their_workspace_until_the_launch(cuda, monkeypatch, n):
    import weakref

    from slime_amd import optim

    refs, workspace, launch = [], optim._List.workspace, optim._launch
    monkeypatch.setattr(optim._List, "workspace", lambda *a: refs.append(weakref.ref(t := workspace(*a))) or t)
    monkeypatch.setattr(optim, "_launch", lambda *a: launch(*a) if refs[-1]() is not None else pytest.fail("the workspace is gone"))
    ps = [torch.nn.Parameter(torch.zeros(50, device=cuda)) for _ in range(n)]
    for p in ps:
        p.grad = torch.ones(50, device=cuda)
    assert abs(slime_amd.clip_grad_norm_(ps, 1.0).item() - math.sqrt(50 * n)) < 1e-4 and len(refs) == 1
    assert abs(slime_amd.get_total_norm(p.grad for p in ps).item() - 1.0) < 1e-4 and len(refs) == 2


def test_clip_matches_torch(cuda):
    ps = [torch.nn.Parameter(torch.randn(s, device=cuda)) for s in ((64, 64), (100,), (3, 5, 7))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        p.grad, q.grad = p.detach() * 3, q.detach() * 3
    a, b = slime_amd.clip_grad_norm_(ps, 1.0), torch.nn.utils.clip_grad_norm_(qs, 1.0)
    torch.testing.assert_close(a, b, rtol=1e-6, atol=0)
    for p, q in zip(ps, qs):
        torch.testing.assert_close(p.grad, q.grad, rtol=2e-6, atol=0)


# ---- AdamW ----------------------------------------------------------------------------------------------------------------
def adamw_bounds(g, p, m, v, t, c, lr, ls, wd, b1, b2, eps, c_rounds):
    """The step in 64 bits and bounds of its fp32 evaluation's error, a count of roundings each: g' = c g takes c_rounds + 1; a
    fp32 constant one; m: product and constant of b1 m (2), of (1 - b1) g' (that of g' + 1), the last addition (1); v the same
    with (1 - b2) g' g' (twice g' + 2); the root halves v's and adds 1, the constant and the fma with eps 3, the division 1;
    step size (1 / (1 - b1^t), lr and lr_scale) 4; the decay's factor 4 (two constants, two products); two additions into p."""
    g, p, m, v = g.double(), p.double(), m.double(), v.double()
    gs, r = c * g, c_rounds + 1
    m1, v1 = b1 * m + (1 - b1) * gs, b2 * v + (1 - b2) * gs * gs
    em = U * (2 * (b1 * m).abs() + (r + 1) * ((1 - b1) * gs).abs() + m1.abs()) + 2.0 ** -148
    ev = U * (2 * b2 * v + (2 * r + 2) * (1 - b2) * gs * gs + v1) + 2.0 ** -147
    denom = torch.sqrt(v1 / (1 - b2 ** t)) + eps
    step = lr * ls / (1 - b1 ** t)
    upd = step * m1 / denom
    ed = ev / v1.clamp(min=2.0 ** -140) / 2 + 4 * U
    p1 = p - lr * ls * wd * p
    p2 = p1 - upd
    ep = (step / denom) * em + upd.abs() * (ed + 6 * U) + 4 * U * (lr * ls * wd * p).abs() + U * (p1.abs() + p2.abs()) + 2.0 ** -148
    return (p2, ep * 1.01), (m1, em * 1.01), (v1, ev * 1.01)


def near(x, want, bound):
    err = (x.double() - want).abs()
    assert bool((err <= bound).all()), ((err - bound).max().item(), x.shape)


def check_weight(w, want, bound):
    near(w, want, bound + (want.abs() + bound) * torch.finfo(w.dtype).eps / 2 * 1.001 + SUBNORMAL[w.dtype] / 2)


def adamw_case(shapes, g_dtypes, w_dtypes, seed=0, offset=0):
    n = len(shapes)
    p, m = tensors(shapes, [F32], seed, 0.05, offset), tensors(shapes, [F32], seed + 1, 0.02, offset)
    v, g = tensors(shapes, [F32], seed + 2, 0.02, offset), tensors(shapes, g_dtypes, seed + 3, 0.03, offset)
    for x in v:
        x.square_()
    w = [None if w_dtypes[i % len(w_dtypes)] is None else tensors([s], [w_dtypes[i % len(w_dtypes)]], seed + 4, 1.0, offset)[0] for i, s in enumerate(shapes)]
    return p, m, v, g, w, n


@pytest.mark.parametrize("g_dtypes,w_dtypes", [([BF16], [BF16]), ([F32], [BF16]), ([F16], [F16]), ([F32], [None]), ([F32, BF16, F16], [None, F16, BF16])])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("clip", [False, True])
def test_adamw(cuda, g_dtypes, w_dtypes, offset, clip):
    p, m, v, g, w, n = adamw_case(SIZES, g_dtypes, w_dtypes, 20, offset)
    b1, b2, eps, lr, scale = 0.9, 0.95, 1e-8, 3e-3, 0.25
    decay, mult = [0.1 * (i % 3) for i in range(n)], [1.0 + 0.5 * (i % 2) for i in range(n)]
    plan = slime_amd.AdamWPlan(p, g, w, m, v, betas=(b1, b2), eps=eps, weight_decay=decay, lr_scale=mult, step=4)
    assert plan.exp_avgs == m and plan.exp_avg_sqs == v
    for t in (5, 6, 7):
        old = [[x.clone() for x in xs] for xs in (p, m, v)]
        max_norm = 0.4 * norm_of(g) * scale if clip else None
        total = plan.run(lr, max_norm=max_norm, grad_scale=scale)
        c = scale
        if clip:
            check_norm(total, g, scale=scale)
            c *= max_norm / (norm_of(g) * scale + 1e-6)
        else:
            assert total is None
        for i in range(n):
            want = adamw_bounds(g[i], old[0][i], old[1][i], old[2][i], t, c, lr, mult[i], decay[i], b1, b2, eps, 5 if clip else 0)
            for x, (val, bound) in zip((p[i], m[i], v[i]), want):
                near(x, val, bound)
            if w[i] is not None:
                assert torch.equal(w[i], p[i].to(w[i].dtype))           # the copy is the new weight, rounded once
        assert plan.step.item() == t
        for x in g:
            x.mul_(-0.7)
    check_guards(p + m + v + g + [x for x in w if x is not None])


def test_adamw_from_fresh_state_follows_torch(cuda):
    shapes = [(64, 48), (100,), (17, 33)]
    ref = [torch.nn.Parameter(torch.randn(s, device=cuda) * 0.1) for s in shapes]
    ours = [torch.nn.Parameter(r.detach().clone()) for r in ref]
    for x in ref + ours:
        x.grad = torch.zeros_like(x)
    opt = torch.optim.AdamW(ref, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    plan = slime_amd.AdamWPlan(ours, [x.grad for x in ours], betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    for k in range(10):
        for r, o in zip(ref, ours):
            r.grad.normal_()
            o.grad.copy_(r.grad)
        version = ours[0]._version
        opt.step()
        plan.run(1e-2)
        assert ours[0]._version > version                 # autograd hears of the write
        for r, o in zip(ref, ours):
            torch.testing.assert_close(o, r, rtol=0, atol=(k + 1) * 1e-2 * 64 * U + 1e-7)
    assert plan.step.item() == 10


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.0, 0.0), (0.5, 0.0), (0.9999999, 0.99999999)])
@pytest.mark.parametrize("step", [0, 1, 99, 123456789])
def test_adamw_bias_corrections(cuda, betas, step):
    """Early, late and degenerate corrections, which the device forms in 64 bits: the first moment's is seen in the step of an
    element whose moments are steady."""
    b1, b2 = betas
    p, m, v, g = ([torch.full((9,), x, device=cuda)] for x in (0.0, 0.5, 0.25, 0.5))
    plan = slime_amd.AdamWPlan(p, g, None, m, v, betas=betas, eps=0.0, weight_decay=0.0, step=step)
    plan.run(1.0)
    t = step + 1
    want = -(1 - b2 ** t) ** 0.5 / (1 - b1 ** t)
    # fp32 (1 - beta) is exact to u of its own size; moments, root, division and the two step constants: under 16 roundings
    assert abs(p[0][0].item() - want) <= 16 * U * abs(want), (p[0][0].item(), want)
    assert plan.step.item() == t


def test_adamw_zero_gradients_and_state(cuda):
    p = torch.randn(ITEM + 9, device=cuda)
    g = torch.zeros_like(p)
    before = p.clone()
    plan = slime_amd.AdamWPlan([p], [g], weight_decay=0.0)
    assert plan.run(0.1, max_norm=1.0).item() == 0.0
    assert torch.equal(p, before)
    g.fill_(1e-30)                                         # squares vanish: eps keeps the step finite
    plan.run(0.1)
    assert p.isfinite().all()


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_adamw_skips_nonfinite_steps(cuda, norm_type):
    p, m, v, g, w, n = adamw_case([(300, 70), (5,), (2 * ITEM + 1,)], [F16], [F16], 30)
    plan = slime_amd.AdamWPlan(p, g, w, m, v, norm_type=norm_type, skip_nonfinite=True, step=2)
    everything = p + m + v + w
    for bad in (math.inf, -math.inf, math.nan):
        old, good = [x.clone() for x in everything], g[2][-1].clone()
        g[2][-1] = bad
        total = plan.run(1e-3)
        assert not math.isfinite(total.item()) and plan.step.item() == 2
        plan.run(1e-3, max_norm=1.0)
        assert all(torch.equal(a, b) for a, b in zip(everything, old))
        g[2][-1] = good
    check_norm(plan.run(1e-3), g, norm_type)
    assert plan.step.item() == 3 and not torch.equal(p[0], old[0])
    # a norm that was reduced elsewhere decides too
    old = [x.clone() for x in everything]
    given = torch.tensor(math.inf, device=cuda)
    assert plan.run(1e-3, total_norm=given) is given
    assert plan.step.item() == 3 and all(torch.equal(a, b) for a, b in zip(everything, old))


def test_adamw_device_scalars_and_given_norm(cuda):
    shapes = [(33, 65), (ITEM + 4,)]
    a, b = adamw_case(shapes, [BF16], [BF16], 40), adamw_case(shapes, [BF16], [BF16], 40)
    pa = slime_amd.AdamWPlan(a[0], a[3], a[4], a[1], a[2])
    pb = slime_amd.AdamWPlan(b[0], b[3], b[4], b[1], b[2])
    lr, scale = torch.tensor(2.0 ** -9, device=cuda), torch.tensor([0.125], device=cuda)
    norm = slime_amd.GradNormPlan(a[3]).run(grad_scale=0.125).clone()
    pa.run(2.0 ** -9, max_norm=0.5, grad_scale=0.125)
    assert pb.run(lr, max_norm=0.5, grad_scale=scale, total_norm=norm) is norm
    for xs, ys in zip(a[:3] + (a[4],), b[:3] + (b[4],)):
        assert all(torch.equal(x, y) for x, y in zip(xs, ys))
    with pytest.raises(ValueError, match="lr"):
        pa.run(torch.tensor(0.1))
    for call in (lambda: pa.run(0.1, grad_scale=pa.total_norm), lambda: pa.run(pa.total_norm)):
        with pytest.raises(ValueError, match="own total_norm"):
            call()
    for plan in (slime_amd.GradNormPlan(a[3]), slime_amd.GradClipPlan(a[3])):
        with pytest.raises(ValueError, match="own total_norm"):
            plan.run(*([1.0] if isinstance(plan, slime_amd.GradClipPlan) else []), grad_scale=plan.total_norm)


def test_adamw_any_dense_layout_and_fresh_moments(cuda):
    p = [torch.randn(8, 6, 4, device=cuda).permute(2, 0, 1), torch.randn(5, 1, device=cuda)]
    g = [torch.empty_strided(x.shape, x.stride(), device=cuda).normal_() for x in p]
    old = [x.clone() for x in p]
    plan = slime_amd.AdamWPlan(p, g, weight_decay=0.0, eps=0.0)
    plan.run(0.01)
    for x, o, y in zip(p, old, g):
        torch.testing.assert_close(x, o - 0.01 * y.sign(), rtol=0, atol=1e-6)


# ---- random lists ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(24))
def test_random_lists(cuda, seed):
    """Lists of random lengths, sizes (around the pieces too), types and starts through all forms, in one packed buffer per role as
    trainers hold them; what lies between the tensors stays."""
    import random

    rng = random.Random(1000 + seed)
    n = rng.choice([1, 2, 7, 40, 200])
    base = [1, 3, 255, 1023, 4096, 8192, ITEM, 2 * ITEM]
    sizes = [max(0, rng.choice(base) * rng.choice([1, 1, 2]) + rng.randint(-3, 3)) if rng.random() < 0.7 else rng.randint(0, 40000) for _ in range(n)]
    norm_type = rng.choice([2.0, 2.0, math.inf])

    def packed(dtype, scale):
        gaps = [rng.choice([0, 0, 1, 2, 7, 64]) for _ in range(n + 1)]
        total = sum(sizes) + sum(gaps)
        buf = torch.full((total,), 7.0, dtype=dtype, device=cuda)
        keep = torch.ones(total, dtype=torch.bool, device=cuda)
        views, at = [], gaps[0]
        for i, k in enumerate(sizes):
            v = buf[at:at + k]
            v.normal_().mul_(scale)
            keep[at:at + k] = False
            views.append(v)
            at += k + gaps[i + 1]
        return views, lambda: bool((buf[keep] == 7).all())

    gd, od, wd = rng.choice([BF16, F16, F32]), rng.choice([BF16, F16, F32]), rng.choice([None, BF16, F16])
    (g, g_ok), (o, o_ok) = packed(gd, 0.05), packed(od, 1.0)
    ref = norm_of(g, norm_type)
    check_norm(slime_amd.get_total_norm(g, norm_type), g, norm_type)
    total, each = slime_amd.GradNormPlan(g, norm_type, per_tensor=True).run()
    check_norm(total, g, norm_type)
    for e, t in zip(each, g):
        check_norm(e, [t], norm_type)
    before = [t.clone() for t in g]
    max_norm, scale = ref * rng.choice([0.3, 0.9, 2.0]) + 1e-3, rng.choice([1.0, 0.5, 0.01])
    slime_amd.GradClipPlan(g, norm_type, out=o).run(max_norm * scale, grad_scale=scale)
    check_clip(o, before, max_norm * scale, ref * scale, scale)
    assert all(torch.equal(a, b) for a, b in zip(g, before))
    if rng.random() < 0.5:
        slime_amd.GradClipPlan(g, norm_type).run(max_norm)
    else:
        ps = [torch.nn.Parameter(torch.empty_like(t)) for t in g]
        for p, t in zip(ps, g):
            p.grad = t
        slime_amd.clip_grad_norm_(ps, max_norm, norm_type)
    check_clip(g, before, max_norm, ref)
    (p, p_ok), (m, m_ok), (v, v_ok) = packed(F32, 0.05), packed(F32, 0.02), packed(F32, 0.02)
    w, w_ok = packed(wd, 1.0) if wd else ([None] * n, lambda: True)
    for x in v:
        x.square_()
    old, ref = [[x.clone() for x in xs] for xs in (p, m, v)], norm_of(g, norm_type)
    clip = rng.random() < 0.7
    plan = slime_amd.AdamWPlan(p, g, w, m, v, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.2, norm_type=norm_type, step=3)
    plan.run(1e-2, max_norm=max_norm * scale if clip else None, grad_scale=scale)
    c = scale * (min(1.0, max_norm * scale / (ref * scale + 1e-6)) if clip else 1.0)
    for i in range(n):
        want = adamw_bounds(g[i], old[0][i], old[1][i], old[2][i], 4, c, 1e-2, 1.0, 0.2, 0.8, 0.99, 1e-6, 5)
        for x, (val, bound) in zip((p[i], m[i], v[i]), want):
            near(x, val, bound)
        if wd:
            assert torch.equal(w[i], p[i].to(wd))
    assert all(ok() for ok in (g_ok, o_ok, p_ok, m_ok, v_ok, w_ok))


# ---- streams, graphs, and the run of them together ------------------------------------------------------------------------
def test_plans_run_on_another_stream(cuda):
    ts = tensors([(1000, 999)] * 3, [BF16], 50)
    side = torch.cuda.Stream()
    plan, norm = slime_amd.GradClipPlan(ts), slime_amd.GradNormPlan(ts)
    before = [t.clone() for t in ts]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n = norm.run().clone()
        plan.run(1.0)
        p = torch.nn.Parameter(torch.zeros(1000, 999, dtype=BF16, device=cuda))
        p.grad = ts[0]
        m = slime_amd.clip_grad_norm_(p, 0.25)
    side.synchronize()
    check_norm(n, before)
    check_clip(ts[1:], before[1:], 1.0, norm_of(before))
    assert abs(norm_of([ts[0]]) - 0.25) < 1e-3 and m.item() > 0.5


def test_functions_in_a_graph(cuda):
    ts = tensors([(5,)] * 200, [F32, BF16], 51)
    p = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    for q, t in zip(p, ts):
        q.grad = t
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm = slime_amd.get_total_norm(ts)
            total = slime_amd.clip_grad_norm_(p, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        for i, t in enumerate(ts):
            t.normal_().mul_(1 + (i + k) % 3)
        before = [t.clone() for t in ts]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_norm(norm, before)
        assert torch.equal(norm, total)
        check_clip(ts, before, 1.0, norm_of(before))


def test_a_training_step_as_it_is_used(cuda):
    """Straight-through INT4 forward, backward, norm of every tensor, clipped update, block-FP8 of the new weights - eagerly and
    replayed from a graph, step for step the same bits."""
    shapes = [(256, 384), (128, 256), (384, 128)]

    def build():
        gen = torch.Generator().manual_seed(60)
        master = [(torch.randn(s, generator=gen) * 0.05).to(cuda) for s in shapes]
        weight = [x.to(BF16).requires_grad_() for x in master]
        main = [torch.zeros_like(x) for x in master]
        grads = [torch.zeros_like(x) for x in weight]
        return {"master": master, "weight": weight, "main": main, "grads": grads, "norm": slime_amd.GradNormPlan(grads, per_tensor=True),
                "clip": slime_amd.GradClipPlan(grads, out=main),
                "adamw": slime_amd.AdamWPlan(master, main, [w.detach() for w in weight], weight_decay=0.1),
                "fp8": slime_amd.Fp8QuantPlan([w.detach() for w in weight], (128, 128), mode=1)}

    def backward(s, k):
        gen = torch.Generator().manual_seed(70 + k)
        for w, g in zip(s["weight"], s["grads"]):
            x = torch.randn(w.shape[1], 64, generator=gen).to(cuda, BF16)
            y = slime_amd.fake_int4_quantization_ste(w, 128) @ x
            g.copy_(torch.autograd.grad(y.float().square().sum(), w)[0])

    def step(s):
        s["norm"].run()
        total = s["clip"].run(1.0)
        s["adamw"].run(1e-2)
        s["fp8"].run()
        return total

    eager, played = build(), build()
    backward(played, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(played)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        backward(eager, k)
        backward(played, k)
        total = step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert total.item() > 1.0 and torch.equal(total, eager["norm"].total_norm)
        check_norm(total, eager["grads"])
        check_clip(eager["main"], eager["grads"], 1.0, norm_of(eager["grads"]))
        assert abs(norm_of(eager["main"]) - 1.0) < 1e-5
        for name in ("master", "weight", "main"):
            assert all(torch.equal(a, b) for a, b in zip(eager[name], played[name])), (k, name)
        assert torch.equal(eager["norm"].norms, played["norm"].norms)
        assert eager["adamw"].step.item() == played["adamw"].step.item() == k + 1
        for w, (q, sc), (q2, sc2) in zip(eager["weight"], eager["fp8"].outputs, played["fp8"].outputs):
            qe, se = slime_amd.blockwise_cast_to_fp8_triton(w.detach(), (128, 128))
            assert torch.equal(q.view(torch.uint8), qe.view(torch.uint8)) and torch.equal(sc, se)
            assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(sc, sc2)


def test_inference_tensors_and_saved_tensors(cuda):
    """Tensors without a version counter work; autograd refuses a backward through what a clip has overwritten."""
    with torch.inference_mode():
        t = torch.ones(100, device=cuda)
        p = torch.nn.Parameter(torch.zeros(100, device=cuda), requires_grad=False)
    p.grad = t
    assert abs(slime_amd.clip_grad_norm_(p, 1.0).item() - 10.0) < 1e-5 and abs(t[0].item() - 0.1) < 1e-6
    slime_amd.GradClipPlan([t]).run(0.5)
    assert abs(t[0].item() - 0.05) < 1e-6
    x = torch.ones(10, device=cuda, requires_grad=True)
    g = torch.full((10,), 3.0, device=cuda)
    y = (x * g).sum()                                       # saves g
    slime_amd.GradClipPlan([g]).run(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_calls_from_two_threads_on_streams_of_their_own(cuda):
    import threading

    lists = [tensors([(1000, 37 + i), (5,), (ITEM * 3 + i,)] * 20, [BF16, F32], 80 + i, 1.0 + i) for i in range(2)]
    want = [norm_of(ts) for ts in lists]
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            plan = slime_amd.GradNormPlan(lists[i], per_tensor=True)
            for k in range(30):
                a, b = slime_amd.get_total_norm(lists[i]), plan.run()[0]
                if abs(a.item() - want[i]) > 2 * U * want[i] or abs(b.item() - want[i]) > 2 * U * want[i]:
                    bad.append((i, k, a.item(), b.item()))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_two_graphs_of_one_plan_replayed_in_turn(cuda):
    ts = tensors([(ITEM * 2 + 3,), (77, 5)], [BF16], 90)
    norm, clip = slime_amd.GradNormPlan(ts), slime_amd.GradClipPlan(ts)
    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for max_norm in (3.0, 1.0):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.stream(side), torch.cuda.graph(graphs[-1], stream=side):
            norm.run()
            clip.run(max_norm)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        for t in ts:
            t.normal_()
        before = [t.clone() for t in ts]
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert abs(norm.total_norm.item() - 3.0) < 1e-2 and abs(norm_of(ts) - 1.0) < 1e-2       # bf16 roundings average out
        assert all(((t.double() - b.double() / norm_of(before)).abs() <= b.double().abs() / norm_of(before) * 2.0 ** -6).all() for t, b in zip(ts, before))


def test_item_tables_are_exact(cuda):
    """Every row of a table of half a million pieces, from tensors of mixed types and starts (a per-lane 64-bit shift went wrong in
    one wavefront of a hundred here)."""
    import numpy as np

    from slime_amd import optim

    rng = np.random.default_rng(1)
    base, rows = 0x7F0000000000, []
    for i in range(400):
        g, o = int(rng.integers(0, 3)), int(rng.integers(0, 3))
        rows.append([base + 64 * i * 4, base + (1 << 40) + 2 * 64 * i + 4 * i, int(rng.integers(1, 20_000_000)) if i else (1 << 31) + 12345, g | o << 32])
    for words in (4, 8):
        if words == 8:
            rows = [r + [base + (2 << 40) + 4 * i, base + (3 << 40), base + (4 << 40), i] for i, r in enumerate(rows)]
        table = np.array(rows, dtype=np.int64)
        items, starts, n = optim._item_table(table, cuda, "test")
        got, starts = items.cpu().numpy(), starts.cpu().numpy()
        owner = np.repeat(np.arange(len(rows)), np.diff(starts))
        per, phase = (np.broadcast_to(x, len(rows))[owner] for x in optim._cuts(table))
        piece, src = np.arange(n) - starts[owner], table[owner]
        at = np.where(piece > 0, piece * per - phase, 0)
        g, o = (np.where(d == 1, 4, 2) for d in (src[:, 3] & 0xFFFFFFFF, src[:, 3] >> 32))
        assert n > 300_000 and np.array_equal(got[:, 0], src[:, 0] + at * g) and np.array_equal(got[:, 1], src[:, 1] + at * o)
        assert np.array_equal(got[:, 2], np.minimum((piece + 1) * per - phase, src[:, 2]) - at) and np.array_equal(got[:, 3], src[:, 3])
        assert (np.add.reduceat(got[:, 2], starts[:-1]) == table[:, 2]).all()
        for w in range(4, words):
            assert np.array_equal(got[:, w], src[:, w] + (at * 4 if w < 7 else 0))


def test_a_list_of_more_than_four_gigabytes(cuda):
    """Offsets past 32 bits, in one tensor and over the list."""
    n = (1 << 31) + 12345
    big = torch.zeros(n, dtype=BF16, device=cuda)
    small = torch.full((77,), 3.0, dtype=F32, device=cuda)
    at = torch.tensor([0, 1 << 30, (1 << 31) - 1, 1 << 31, n - 1], device=cuda)
    big[at] = 4.0
    want = math.sqrt(5 * 16.0 + 77 * 9.0)
    plan = slime_amd.GradClipPlan([big, small])
    total = plan.run(want / 2)
    assert abs(total.item() - want) <= 2 * U * want
    assert big[at].tolist() == [2.0] * 5 and big.count_nonzero().item() == 5
    assert (small - 1.5).abs().max().item() < 1e-6


def test_abi_constants_match(cuda):
    assert _lib.GRAD_ITEM_BYTES == ITEM and 2 * _lib.ADAMW_ITEM == ITEM


# ---- device scalars that lie in tensors of the call -----------------------------------------------------------------------
def test_scalars_inside_tensors_of_a_plan(cuda):
    """A scale among the gradients that a plan only reads is an ordinary value; one that its run writes is refused; an AdamW run
    has read its scalars before it writes."""
    g = tensors([(3 * ITEM + 5,), (4,), (300, 520)], [F32], 100, 0.2)
    g[1][2] = 0.37
    plan = slime_amd.GradNormPlan(g, per_tensor=True)
    total, each = plan.run(grad_scale=g[1][2])
    check_norm(total, g, scale=g[1][2].item())
    for bad in plan.norms:
        with pytest.raises(ValueError, match="must not lie in"):
            plan.run(grad_scale=bad)
    clip = slime_amd.GradClipPlan(g)
    with pytest.raises(ValueError, match="must not lie in"):
        clip.run(1.0, grad_scale=g[1][2])
    with pytest.raises(ValueError, match="must not lie in"):
        clip.run(1.0, total_norm=g[0][5])
    a, b = (adamw_case([(2 * ITEM + 1,), (5,)], [BF16], [BF16], 101) for _ in range(2))
    for x in (a, b):
        x[0][1][3], x[0][1][4] = 2.0 ** -9, 0.125
    pa, pb = (slime_amd.AdamWPlan(x[0], x[3], x[4], x[1], x[2]) for x in (a, b))
    pa.run(2.0 ** -9, max_norm=0.5, grad_scale=0.125)
    pb.run(b[0][1][3], max_norm=0.5, grad_scale=b[0][1][4])
    for xs, ys in zip(a[:3] + (a[4],), b[:3] + (b[4],)):
        assert all(torch.equal(x, y) for x, y in zip(xs, ys))


@pytest.mark.parametrize("n", [1, 3, 200])
def test_clip_by_a_norm_that_is_among_the_gradients(cuda, n):
    """The norm as it is at the call, as torch has it, in all launches of a long list."""
    ts = tensors([(3 * ITEM + 5,)] + [(5,)] * (n - 1), [F32], 102)
    ts[0][7] = 50.0
    before = [t.clone() for t in ts]
    ps = [torch.nn.Parameter(torch.empty_like(t)) for t in ts]
    for p, t in zip(ps, ts):
        p.grad = t
    slime_amd.clip_grads_with_norm_(ps, 2.0, ts[0][7])
    check_clip(ts, before, 2.0, 50.0)
    check_guards(ts)


# ---- the C entry points -----------------------------------------------------------------------------------------------------
def test_workspaces_of_sixteen_byte_alignment(cuda):
    """All entry points on a workspace that is aligned to 16 bytes and to no more."""
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    a, b = (adamw_case([(2 * ITEM + 1,), (5,)], [BF16], [BF16], 110) for _ in range(2))
    plan = slime_amd.AdamWPlan(a[0], a[3], a[4], a[1], a[2])
    plan.run(1e-2, max_norm=0.5, grad_scale=0.25)
    other = slime_amd.AdamWPlan(b[0], b[3], b[4], b[1], b[2])
    room = torch.zeros(lib.wq_grad_workspace_bytes(other._n_items) // 8 + 2, dtype=torch.int64, device=cuda)
    h = other._hyper
    h.lr, h.max_norm, h.grad_scale = 1e-2, 0.5, 0.25
    assert room.data_ptr() % 32 == 0
    assert lib.wq_adamw_items(other._items.data_ptr(), other._n_items, h, room.data_ptr() + 16, st) == 0
    assert torch.equal(plan.total_norm, other.total_norm)
    for xs, ys in zip(a[:3] + (a[4],), b[:3] + (b[4],)):
        assert all(torch.equal(x, y) for x, y in zip(xs, ys))
    total = torch.zeros((), device=cuda)
    assert lib.wq_grad_norm_items(other._items.data_ptr(), other._n_items, 8, None, 0, 0, 0.25, None, room.data_ptr() + 16, total.data_ptr(),
                                  None, st) == 0
    assert torch.equal(total, plan.total_norm) and room[0].item() == 0 and room[1].item() == 0


# ---- lists whose partials are folded in two levels ----------------------------------------------------------------------------
FOLD_GROUP, FOLD_DIRECT = 4096, 8 * 4096


@pytest.fixture(autouse=True)
def seeded(request):
    """What a test draws on the device is the same on each run of it."""
    import zlib

    torch.manual_seed(zlib.crc32(request.node.name.encode()))


def long_list(pieces, dtype, device):
    """Tensors of so many pieces in all, the first one nearly all of them; non-zero everywhere."""
    item = ITEM // torch.empty((), dtype=dtype).element_size()
    buf = torch.empty(pieces * item, dtype=dtype, device=device).normal_()
    buf[buf == 0] = 1
    cuts = [0, (pieces - 41) * item] + [(pieces - 40 + i) * item for i in range(41)]
    return buf, [buf[a:b] for a, b in zip(cuts, cuts[1:])]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pieces", [FOLD_DIRECT, FOLD_DIRECT + 1, FOLD_DIRECT + 3 * FOLD_GROUP + 1000])
def test_long_norms(cuda, pieces, dtype):
    buf, ts = long_list(pieces, dtype, cuda)
    plans = {k: slime_amd.GradNormPlan(ts, k, per_tensor=True) for k in (2.0, math.inf)}
    assert plans[2.0]._n_items == pieces
    for k, plan in plans.items():
        total, each = plan.run()
        check_norm(total, ts, k)
        check_norm(slime_amd.get_total_norm(ts, k), ts, k)
        check_norm(plan.run(grad_scale=0.37)[0], ts, k, float(torch.tensor(0.37)))
        plan.run()
        for e, t in zip(each, ts):
            check_norm(e, [t], k)
    # every group of partials counts: a value that stands out in each in turn, at the first and the last place of it
    item, groups = buf.numel() // pieces, -(-pieces // FOLD_GROUP)
    rest = norm_of([buf])
    for group in range(groups):
        for at in (group * FOLD_GROUP * item, min((group + 1) * FOLD_GROUP, pieces) * item - 1):
            old = buf[at].clone()
            buf[at] = 65536.0
            want = math.sqrt(rest ** 2 - old.double().item() ** 2 + 2.0 ** 32)
            assert plans[math.inf].run()[0].item() == 65536.0 == slime_amd.get_total_norm(ts, math.inf).item()
            assert abs(plans[2.0].run()[0].item() - want) <= 2 * U * want
            buf[at] = math.nan
            assert all(math.isnan(p.run()[0].item()) for p in plans.values())
            buf[at] = old


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_long_clips(cuda, norm_type, dtype):
    buf, ts = long_list(FOLD_DIRECT + 2 * FOLD_GROUP + 77, dtype, cuda)
    before = buf.clone()
    norm = norm_of([before], norm_type)
    check_norm(slime_amd.GradClipPlan(ts, norm_type).run(0.3 * norm), [before], norm_type)
    check_clip([buf], [before], 0.3 * norm, norm)
    buf.copy_(before)
    ps = [torch.nn.Parameter(t.new_empty(t.shape)) for t in ts]
    for p, t in zip(ps, ts):
        p.grad = t
    check_norm(slime_amd.clip_grad_norm_(ps, 0.3 * norm, norm_type), [before], norm_type)
    check_clip([buf], [before], 0.3 * norm, norm)


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("pieces", [FOLD_DIRECT, FOLD_DIRECT + FOLD_GROUP + 5])
def test_long_updates(cuda, norm_type, pieces):
    """The folded sums feed the step's scalars; on both sides of the limit for plain loads, too."""
    n = pieces * _lib.ADAMW_ITEM
    g = torch.empty(n, dtype=BF16, device=cuda).normal_()
    p, m, v = (torch.zeros(n, device=cuda) for _ in range(3))
    cut = n - 3 * _lib.ADAMW_ITEM
    plan = slime_amd.AdamWPlan(*([x[:cut], x[cut:]] for x in (p, g)), exp_avgs=[m[:cut], m[cut:]], exp_avg_sqs=[v[:cut], v[cut:]],
                               norm_type=norm_type, skip_nonfinite=True, weight_decay=0.0)
    assert plan._n_items == pieces
    norm = norm_of([g], norm_type)
    check_norm(plan.run(1e-2, max_norm=0.5 * norm), [g], norm_type)
    c = 0.5 * norm / (norm + 1e-6)
    for a in range(0, n, 1 << 25):
        s = slice(a, min(a + (1 << 25), n))
        zero = torch.zeros(s.stop - a, device=cuda)
        want = adamw_bounds(g[s], zero, zero, zero, 1, c, 1e-2, 1.0, 0.0, 0.9, 0.999, 1e-8, 5)
        for x, (val, bound) in zip((p[s], m[s], v[s]), want):
            near(x, val, bound)
    old = p.clone()
    for at in (5, FOLD_GROUP * _lib.ADAMW_ITEM * 4 + 1, n - 1):           # a NaN in any group stops the step
        keep = g[at].clone()
        g[at] = math.nan
        assert math.isnan(plan.run(1e-2).item()) and plan.step.item() == 1 and torch.equal(p, old)
        g[at] = keep


# ---- norms over ranks ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [1.0, 1e23, 1e-28])
def test_norms_of_parts_reduced_as_over_ranks(cuda, scale):
    """Two lists stand for two ranks' parts; the reductions are those that the module gives, without the collective."""
    parts = [tensors(SIZES, [F32], 120 + i, scale) for i in range(2)]
    both = parts[0] + parts[1]
    before = [[t.clone() for t in ts] for ts in parts]
    squares = [slime_amd.GradNormPlan(ts).run().double().square() for ts in parts]
    total = (squares[0] + squares[1]).sqrt().float()
    want = norm_of(both)
    assert abs(total.item() - want) <= 3 * U * want                         # each part's rounding, and the last one
    for ts, old in zip(parts, before):
        slime_amd.GradClipPlan(ts).run(0.25 * want, total_norm=total)
        c = 0.25 * want / (want + 1e-6)
        for t, o in zip(ts, old):                                          # a coefficient's 6 u, and 2 more of the norm
            assert bool(((t.double() - o.double() * c).abs() <= o.double().abs() * c * 8.01 * U + SUBNORMAL[F32]).all())
    biggest = [slime_amd.GradNormPlan(ts, math.inf).run() for ts in before]
    largest = torch.maximum(*(b.view(torch.int32) for b in biggest)).view(F32)
    check_norm(largest, before[0] + before[1], math.inf)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_the_bits_of_an_infinity_norm_order_like_it(cuda, dtype):
    """NaN above infinity above the rest, as integers: whatever the sign and payload of the NaN, and for infinity times 0."""
    x = torch.zeros(100, dtype=dtype, device=cuda)
    plan = slime_amd.GradNormPlan([x], math.inf)
    inf = int(torch.tensor(math.inf).view(torch.int32))
    for bad in (math.nan, -math.nan):
        x[3] = bad
        for scale in (1.0, 0.5, torch.tensor(-2.0, device=cuda)):
            assert plan.run(scale).view(torch.int32).item() > inf
    if dtype == F32:
        for bits in (0x7F800001, -1, -0x7FFFFF, 0x7FFFFFFF):
            x.view(torch.int32)[3] = bits
            assert plan.run().view(torch.int32).item() > inf and plan.run(0.5).view(torch.int32).item() > inf
    x[3] = -math.inf
    assert plan.run().view(torch.int32).item() == inf
    assert plan.run(0.0).view(torch.int32).item() > inf
    x[3] = 1.0
    assert 0 < plan.run().view(torch.int32).item() < inf
