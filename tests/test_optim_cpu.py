"""Refusals and host logic of the gradient norm, the clip and the AdamW update (no GPU needed: everything here is decided
before a launch)."""

import ctypes
import math

import numpy as np
import pytest
import torch

import slime_amd
from slime_amd import _lib, optim

S, M_, N_ = -2, -3, -1
P = ctypes.c_void_p(64)      # a pointer that is never followed


def _lists(n=3, dtype=torch.float32, shape=(4, 8)):
    return [torch.zeros(shape, dtype=dtype) for _ in range(n)]


# ---- C ABI ---------------------------------------------------------------------------------------------------------------
def test_entry_points_reject_bad_arguments():
    lib = _lib.load()
    assert lib.wq_grad_workspace_bytes(-1) == 0 and lib.wq_grad_workspace_bytes(0) >= 64
    assert lib.wq_grad_workspace_bytes(1000) >= 8000
    assert lib.wq_grad_make_items(None, None, 1, -1, 4, None, None) == S
    assert lib.wq_grad_make_items(None, None, 1, 3, 5, None, None) == S
    assert lib.wq_grad_make_items(None, None, 0, 3, 4, None, None) == S
    assert lib.wq_grad_make_items(None, None, 1, 3, 4, None, None) == N_
    assert lib.wq_grad_make_items(None, None, 0, 0, 4, None, None) == 0
    assert lib.wq_grad_norm_items(None, -1, 4, None, 0, 0, 1.0, None, P, P, None, None) == S
    assert lib.wq_grad_norm_items(None, 1, 6, None, 0, 0, 1.0, None, P, P, None, None) == S
    assert lib.wq_grad_norm_items(P, 1, 4, None, 0, 2, 1.0, None, P, P, None, None) == M_
    assert lib.wq_grad_norm_items(None, 1, 4, None, 0, 0, 1.0, None, P, P, None, None) == N_
    assert lib.wq_grad_norm_items(P, 1, 4, None, 0, 0, 1.0, None, None, P, None, None) == N_
    assert lib.wq_grad_norm_items(P, 1, 4, None, 0, 0, 1.0, None, P, None, None, None) == N_
    assert lib.wq_grad_norm_items(P, 1, 4, None, 2, 0, 1.0, None, P, P, P, None) == N_          # `each` without the starts
    assert lib.wq_grad_clip_items(None, 2, 0, 1.0, 1.0, None, None, P, P, None) == N_
    assert lib.wq_grad_clip_items(P, 2, 0, 1.0, 1.0, None, None, None, P, None) == N_
    assert lib.wq_grad_clip_items(P, -2, 0, 1.0, 1.0, None, P, None, None, None) == S
    assert lib.wq_grad_clip_items(P, 2, 5, 1.0, 1.0, None, P, None, None, None) == M_
    assert lib.wq_grad_clip_items(None, 0, 0, 1.0, 1.0, None, P, None, None, None) == 0         # nothing to do


class _Host:
    """A host list; pointers are never followed."""

    def __init__(self, g=64, n=5, dtype=_lib.DTYPE_F32, count=1):
        self.keep = [(ctypes.c_int64 * 2)(64, g), (ctypes.c_int64 * 2)(3, n), (ctypes.c_int32 * 2)(_lib.DTYPE_BF16, dtype)]
        self.args = [*self.keep, 2]

    def norm(self, ws=None, total=None, kind=0):
        return _lib.load().wq_grad_norm_list(*self.args, kind, 1.0, ws, total, None)

    def clip(self, given=None, ws=None, total=None, kind=0):
        return _lib.load().wq_grad_clip_list(*self.args, kind, 1.0, 1.0, given, ws, total, None)

    def bytes(self):
        return _lib.load().wq_grad_list_workspace_bytes(*self.args)


def test_host_lists_are_checked():
    lib = _lib.load()
    good = _Host()
    assert good.norm() == good.clip() == good.norm(ws=P) == good.norm(total=P) == good.clip(total=P) == N_     # nowhere to put it
    assert good.norm(kind=2) == good.clip(kind=-1) == M_
    assert good.bytes() >= 64 + 2 * 8
    for bad, code in ((_Host(n=-1), S), (_Host(dtype=_lib.DTYPE_F64), M_), (_Host(dtype=-1), M_), (_Host(g=0), N_), (_Host(g=66), -5),
                      (_Host(n=(1 << 40) + 1), -6), (_Host(n=1 << 40), 0)):
        if code:
            assert bad.norm(P, P) == bad.clip(P, P, P) == bad.clip(None, P, P) == code and bad.bytes() == 0, code
        else:
            assert bad.bytes() > (1 << 40) // 4096 * 8
    assert _Host(g=0, n=0).bytes() > 0
    for fn, rest in ((lib.wq_grad_norm_list, (0, 1.0, P, P, None)), (lib.wq_grad_clip_list, (0, 1.0, 1.0, None, P, P, None))):
        assert fn(None, None, None, 2, *rest) == N_ and fn(None, None, None, -1, *rest) == S
        assert fn(good.keep[0], None, good.keep[2], 1, *rest) == N_
    assert lib.wq_grad_clip_list(None, None, None, 0, 0, 1.0, 1.0, P, None, None, None) == 0                   # nothing to do


def _hyper(**change):
    h = dict(beta1=0.9, beta2=0.999, eps=1e-8, lr=1e-3, lr_dev=None, grad_scale_dev=None, total_given=None, total=None, step=64,
             grad_scale=1.0, max_norm=-1.0, norm=0, skip_nonfinite=0)
    h.update(change)
    return _lib.AdamWHyper(**h)


def test_adamw_entry_point_rejects_bad_arguments():
    call = lambda h, items=P, n=1, ws=P: _lib.load().wq_adamw_items(items, n, h, ws, None)      # noqa: E731
    assert call(_hyper(), n=-1) == S
    assert call(None) == N_ and call(_hyper(), items=None) == N_ and call(_hyper(), ws=None) == N_ and call(_hyper(step=None)) == N_
    assert call(_hyper(norm=3)) == M_
    for bad in ({"beta1": 1.0}, {"beta1": -0.1}, {"beta2": 1.5}, {"beta2": math.nan}, {"eps": -1.0}, {"eps": math.nan}):
        assert call(_hyper(**bad)) == S, bad
    assert call(_hyper(max_norm=1.0)) == N_ and call(_hyper(skip_nonfinite=1)) == N_            # a norm, and nowhere to put it


def test_structs_match_the_header():
    assert ctypes.sizeof(_lib.AdamWHyper) == 4 * 8 + 5 * 8 + 4 * 4


# ---- Python refusals ------------------------------------------------------------------------------------------------------
PLANS = [lambda g, **k: optim.GradNormPlan(g, **k), lambda g, **k: optim.GradClipPlan(g, **k),
         lambda g, **k: optim.AdamWPlan([torch.zeros(getattr(x, "shape", 1)) for x in g], g, **k)]


@pytest.mark.parametrize("plan", PLANS)
def test_plans_refuse(plan):
    with pytest.raises(RuntimeError, match="GPU"):
        plan(_lists())
    with pytest.raises(ValueError, match="empty"):
        plan([])
    with pytest.raises(ValueError, match="norm_type"):
        plan(_lists(), norm_type=1.0)
    with pytest.raises(TypeError, match="dtype"):
        plan(_lists(dtype=torch.float64))
    with pytest.raises(TypeError, match="dtype"):
        plan(_lists(dtype=torch.int32))
    with pytest.raises(TypeError, match="expected a tensor"):
        plan([None])
    with pytest.raises(TypeError, match="strided"):
        plan([torch.zeros(4, 4).to_sparse()])
    with pytest.raises(ValueError, match="one run"):
        plan([torch.zeros(4, 8)[:, :5]])
    with pytest.raises(ValueError, match="one run"):
        plan([torch.zeros(4, 1).expand(4, 8)])


def test_what_a_plan_cannot_read_as_it_lies():
    neg = torch.zeros(4, 8, dtype=torch.complex64).conj().imag
    flipped = torch._neg_view(torch.zeros(4, 8))
    assert neg.is_neg() and flipped.is_neg()
    for plan in PLANS:
        with pytest.raises(TypeError, match="negation"):
            plan([flipped])
    odd = np.array([[1025, 1024, 4, 0], [1024, 1025, 4, 0], [1026, 1024, 4, 1], [1024, 1026, 4, 1 << 32]], dtype=np.int64)
    for row in odd:
        with pytest.raises(ValueError, match="multiple of its element"):
            optim._item_table(row[None], torch.device("cpu"), "x")
    for k in (4, 5, 6):
        row = np.array([[1024, 0, 4, 0, 1024, 1024, 1024, 0]], dtype=np.int64)
        row[0, k] += 2
        with pytest.raises(ValueError, match="multiple of its element"):
            optim._item_table(row, torch.device("cpu"), "x")


def test_lists_may_be_iterators_and_numbers_numpy_ones():
    with pytest.raises(RuntimeError, match="GPU"):
        optim.AdamWPlan(iter(_lists()), iter(_lists()), iter([None, None, None]), iter(_lists()), iter(_lists()),
                        weight_decay=np.float32(0.1), lr_scale=np.ones(3))
    with pytest.raises(RuntimeError, match="GPU"):
        optim.GradClipPlan(iter(_lists()), out=iter(_lists()))


@pytest.mark.parametrize("call", [lambda g: slime_amd.get_total_norm(g), lambda g: slime_amd.get_total_norm(g[0]),
                                  lambda g: slime_amd.clip_grad_norm_(_params(g), 1.0),
                                  lambda g: slime_amd.clip_grad_norm_(_params(g)[0], 1.0, error_if_nonfinite=True),
                                  lambda g: slime_amd.clip_grads_with_norm_(_params(g), 1.0, torch.ones(()))])
def test_functions_refuse_host_tensors_and_types(call):
    with pytest.raises(RuntimeError, match="GPU"):
        call(_lists())
    with pytest.raises(TypeError, match="dtype"):
        call(_lists(dtype=torch.float64))


def _params(grads):
    ps = [torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


def test_functions_check_their_numbers():
    ps = _params(_lists())
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            slime_amd.clip_grad_norm_(ps, bad)
        with pytest.raises(ValueError, match="max_norm"):
            slime_amd.clip_grads_with_norm_(ps, bad, torch.ones(()))
    with pytest.raises(ValueError, match="norm_type"):
        slime_amd.clip_grad_norm_(ps, 1.0, norm_type=3)
    with pytest.raises(ValueError, match="norm_type"):
        slime_amd.get_total_norm(_lists(), 1)
    with pytest.raises(TypeError, match="total_norm"):
        slime_amd.clip_grads_with_norm_(ps, 1.0, 2.0)


def test_nothing_to_do_needs_no_gpu():
    assert slime_amd.get_total_norm([]).item() == 0.0
    assert slime_amd.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0).item() == 0.0
    assert slime_amd.clip_grad_norm_(iter([]), 1.0).item() == 0.0
    assert slime_amd.clip_grads_with_norm_([], 1.0, torch.ones(())) is None


def test_clip_plan_checks_its_outputs():
    g = _lists()
    with pytest.raises(ValueError, match="one output"):
        optim.GradClipPlan(g, out=_lists(2))
    with pytest.raises(ValueError, match="output of shape"):
        optim.GradClipPlan(g, out=_lists(shape=(8, 4)))
    with pytest.raises(ValueError, match="output of shape"):
        optim.GradClipPlan(g, out=[x.t().contiguous().t() for x in _lists()])
    with pytest.raises(TypeError, match="dtype"):
        optim.GradClipPlan(g, out=_lists(dtype=torch.float64))
    with pytest.raises(ValueError, match="share memory"):
        optim.GradClipPlan([g[0], g[1], g[0]])
    with pytest.raises(ValueError, match="share memory"):
        optim.GradClipPlan(g, out=[g[1], g[0], g[2]])                    # each other's
    buf = torch.zeros(40)
    with pytest.raises(ValueError, match="share memory"):
        optim.GradClipPlan([buf[0:8], buf[16:24]], out=[buf[32:40], buf[30:38]])
    with pytest.raises(RuntimeError, match="GPU"):                        # neighbours, and in place next to apart: fine so far
        optim.GradClipPlan([buf[0:8], buf[8:16]], out=[buf[0:8], buf[16:24]])


def test_adamw_plan_checks_its_lists():
    p, g = _lists(), _lists()
    make = lambda **k: optim.AdamWPlan(p, g, **k)      # noqa: E731
    with pytest.raises(ValueError, match="equally many"):
        optim.AdamWPlan(p, _lists(2))
    with pytest.raises(ValueError, match="equally many"):
        make(weights=_lists(2, torch.bfloat16))
    with pytest.raises(ValueError, match="equally many"):
        make(exp_avgs=_lists(4))
    for bad in ({"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"betas": (math.nan, 0.9)}, {"eps": -1.0}, {"eps": math.nan}):
        with pytest.raises(ValueError, match="betas"):
            make(**bad)
    with pytest.raises(ValueError, match="step"):
        make(step=-1)
    for what in ("weight_decay", "lr_scale"):
        for bad in (-0.1, math.nan, math.inf):
            with pytest.raises(ValueError, match=what):
                make(**{what: bad})
        with pytest.raises(ValueError, match="one " + what):
            make(**{what: [0.1, 0.2]})
    with pytest.raises(TypeError, match="parameters"):
        optim.AdamWPlan(_lists(dtype=torch.bfloat16), g)
    with pytest.raises(TypeError, match="moments"):
        make(exp_avg_sqs=_lists(dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="weights"):
        make(weights=_lists(dtype=torch.float32))
    for other in (_lists(shape=(8, 4)), [x.t().contiguous().t() for x in _lists()]):
        with pytest.raises(ValueError, match="strides of their parameter"):
            optim.AdamWPlan(p, other)
        with pytest.raises(ValueError, match="strides of their parameter"):
            make(exp_avgs=other)
    with pytest.raises(ValueError, match="share memory"):
        make(exp_avgs=g)
    with pytest.raises(ValueError, match="share memory"):
        make(exp_avgs=_lists(), exp_avg_sqs=[p[0]] + _lists(2))
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamWPlan([p[0], p[0]], g[:2])
    with pytest.raises(RuntimeError, match="GPU"):                        # one gradient for two parameters is only read
        optim.AdamWPlan(p, [g[0], g[0], g[1]])
    with pytest.raises(RuntimeError, match="GPU"):
        make(weights=[None, None, torch.zeros(4, 8, dtype=torch.bfloat16)], lr_scale=[1, 2.0, 3], weight_decay=0)


def test_ranges():
    a = torch.zeros(100)
    ok = lambda w, r: optim._refuse_overlaps(w, r, "x")      # noqa: E731
    ok([a[:10], a[10:20]], [a[20:30], a[25:40]])             # what is only read may overlap
    ok([a[10:20], a[:0]], [a[:10], a[15:15], a[20:]])
    for w, r in (([a[:10], a[9:20]], []), ([a[5:6]], [a[:100]]), ([a[:100]], [a[99:]]), ([a[3:7], a[3:7]], []),
                 ([a[50:60]], [a[:55], a[2:4]]), ([a[:4], a[90:95]], [a[10:94]])):
        with pytest.raises(ValueError, match="share memory"):
            ok(w, r)


def test_dense_and_self_overlap():
    x = torch.zeros(4, 6, 5)
    assert all(optim._is_dense(t) for t in (x, x.permute(2, 0, 1), x[1], x[:, :, :0], x[0, 0, 0], x[:1, 2:3].transpose(0, 1)))
    assert not any(optim._is_dense(t) for t in (x[:, :3], x[..., ::2], x[:, 0], x[:1, :1].expand(4, 6, 5)))
    for t in (x[:, :3], x[..., ::2], x.permute(1, 2, 0)[::3]):
        optim._check_no_self_overlap(t, "x")
    for t in (x[:1, :1].expand(4, 6, 5), torch.zeros(9).as_strided((3, 3), (2, 1))):
        with pytest.raises(ValueError, match="share memory"):
            optim._check_no_self_overlap(t, "x")


def test_scalar_arguments():
    dev = torch.device("cpu")
    assert optim._scale_args(0.5, dev, "x") == (0.5, None) and optim._scale_args(2, dev, "x") == (2.0, None)
    t = torch.ones(1)
    assert optim._scale_args(t, dev, "x") == (1.0, t.data_ptr())
    for bad in (-1.0, math.inf, math.nan, torch.ones(2), torch.ones((), dtype=torch.float64)):
        with pytest.raises(ValueError):
            optim._scale_args(bad, dev, "x")


def test_packed_floats_reach_the_descriptor():
    """lr_scale and weight_decay travel as the two halves of one 8-byte word, lr_scale first, as wq_adamw_desc has them."""
    word = np.array([[1.5, 0.25]], dtype=np.float32).view(np.int64)
    assert [ctypes.c_float.from_buffer_copy(word.tobytes()[i:i + 4]).value for i in (0, 4)] == [1.5, 0.25]


def test_pieces_end_at_lines():
    """The host's count of pieces is that of cutting at 128-byte lines of the stream that sets the pace."""
    B, F = _lib.DTYPE_BF16, _lib.DTYPE_F32
    rows = np.array([[128 + 2, 0, 5, B], [256, 256, 8192, B | B << 32], [256 + 2, 256 + 2, 8192, B | B << 32], [256, 512 + 4, 8192, B | F << 32],
                     [256 + 4, 512, 4096, F | B << 32], [256, 512, 0, F | F << 32]], dtype=np.int64)
    per, phase = optim._cuts(rows)
    assert per.tolist() == [8192, 8192, 8192, 8192, 4096, 4096] and phase.tolist() == [1, 0, 1, 1, 1, 0]
    adam = np.array([[64, 0, 9, F, 1024 + 124, 0, 0, 0]], dtype=np.int64)
    per, phase = optim._cuts(adam)
    assert per == _lib.ADAMW_ITEM and phase.tolist() == [31]
    for ptr in range(0, 128, 4):
        for n in (0, 1, 100, 4095, 4096, 4097, 12288):
            host = _Host(g=1024 + ptr, n=n)
            count = 1 + (0 if n == 0 else -(-(n + ptr // 4) // 4096))
            assert host.bytes() == 64 + (count + 1) * 8


def test_no_64_bit_shift_by_a_vector_register(tmp_path):
    """A 64-bit vector shift whose amount is in the last VGPR of a kernel goes wrong now and then on gfx950 (rows of an item
    table came out unshifted), and the register allocator decides which kernel that hits: no kernel has such a shift by a
    VGPR.  Compiles every kernel source with the library's own flags, as the test of flat instructions does."""
    import concurrent.futures
    import glob
    import os
    import re
    import shutil
    import subprocess

    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "slime_amd", "csrc")
    flags = re.search(r"^HIPFLAGS \?= (.*?)\n(?!\s)", open(os.path.join(csrc, "Makefile")).read(), re.S | re.M).group(1)
    flags = flags.replace("\\\n", " ").replace("$(ARCH)", "gfx950").split()

    def shifts(src):
        out = tmp_path / (os.path.basename(src) + ".s")
        subprocess.check_call([hipcc, *flags, "-S", "--cuda-device-only", "-o", str(out), src], stderr=subprocess.DEVNULL)
        text = out.read_text()
        assert "s_endpgm" in text or "wq_api" in src
        return src, re.findall(r"v_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)\S* +\S+ +v\d+,.*", text)

    with concurrent.futures.ThreadPoolExecutor(max_workers=4) as pool:
        for src, found in pool.map(shifts, sorted(glob.glob(os.path.join(csrc, "*.hip")))):
            assert not found, (os.path.basename(src), found)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_list_workspace_is_large_enough(dtype):
    """The bound that the host allocates by against the library's count, wherever the tensors start."""
    size = torch.empty((), dtype=dtype).element_size()
    for shift in range(0, 128, size):
        for sizes in ([1], [4096, 8192], [1] * 300, [40960 * 3 + 1, 0, 7, 5_000_000], [0]):
            n = (ctypes.c_int64 * len(sizes))(*sizes)
            ptr = (ctypes.c_int64 * len(sizes))(*[(1 << 40) + shift] * len(sizes))
            kind = (ctypes.c_int32 * len(sizes))(*[optim._DTYPES[dtype]] * len(sizes))
            need = _lib.load().wq_grad_list_workspace_bytes(ptr, n, kind, len(sizes))
            lst = optim._List.__new__(optim._List)
            lst.n, lst.device = sizes, torch.device("cpu")
            assert 0 < need <= lst.workspace().numel() * 8


def test_list_overlaps():
    for count in (3, 40):                        # the short form and the arrays
        buf = torch.zeros(count * 10 + 10)
        lst = optim._List.__new__(optim._List)

        def check(ts):
            lst.ptr, lst.n = (optim.array("q", [getattr(t, f)() for t in ts]) for f in ("data_ptr", "numel"))
            lst.dtype = optim.array("i", [optim._DTYPES[t.dtype] for t in ts])
            lst._refuse_overlaps("x")

        ts = [buf[10 * i:10 * i + 10] for i in range(count)]
        check(ts[::-1])
        check(ts + [buf[5:5], buf[15:15]])
        for more in (buf[:1], buf[count * 10 - 1:], ts[count // 2], buf):
            with pytest.raises(ValueError, match="share memory"):
                check(ts + [more])


# ---- device scalars --------------------------------------------------------------------------------------------------------
@pytest.fixture
def host_plans(monkeypatch):
    """Plans over host tensors: everything but the tables, the workspace and the launches; -> the launches that were asked for."""
    calls = []

    def build(self, rows, device, what):
        self.device, self._what = device, what
        self.total_norm = torch.zeros((), dtype=torch.float32)
        self._owned, self._n_items = [self.total_norm], 1
        self._items = self._starts = self._workspace = self.total_norm

    monkeypatch.setattr(optim, "_one_device", lambda tensors, what: torch.device("cpu"))
    monkeypatch.setattr(optim._Plan, "_build", build)
    monkeypatch.setattr(optim._Plan, "_built", lambda self: None)
    monkeypatch.setattr(optim._Plan, "_run", lambda self, *args: calls.append(args))
    return calls


def test_plans_refuse_scalars_in_what_they_write(host_plans):
    """The norm of tensor i is written by its workgroup while the others read the scale: a scale there is a race."""
    g = _lists(4)
    plan = optim.GradNormPlan(g, per_tensor=True)
    for scale in (plan.norms[0], plan.norms[3], plan.norms[1:2]):
        with pytest.raises(ValueError, match="grad_scale must not lie in"):
            plan.run(grad_scale=scale)
    with pytest.raises(ValueError, match="own total_norm"):
        plan.run(grad_scale=plan.total_norm)
    plan.run(grad_scale=g[0][0, 0])                                       # gradients are only read here
    assert len(host_plans) == 1
    buf = torch.zeros(100)
    half = torch.zeros(20, dtype=torch.bfloat16)
    plan = optim.GradClipPlan([buf[10:20], buf[30:30], buf[40:41], half[:3]])
    odd = half.view(torch.float32)[1:2]                                   # its first half is written
    for bad in (buf[10], buf[19], buf[40:41], odd):
        with pytest.raises(ValueError, match="grad_scale must not lie in"):
            plan.run(1.0, grad_scale=bad)
        with pytest.raises(ValueError, match="total_norm must not lie in"):
            plan.run(1.0, total_norm=bad)
    for good in (buf[9], buf[20], buf[30], buf[39], buf[41], half.view(torch.float32)[2]):
        plan.run(1.0, grad_scale=good, total_norm=good)
    plan.run(1.0, total_norm=plan.total_norm)                             # not written when a norm is given
    apart = optim.GradClipPlan([buf[0:4]], out=[buf[50:54]])
    apart.run(1.0, grad_scale=buf[0], total_norm=buf[3])
    with pytest.raises(ValueError, match="must not lie in"):
        apart.run(1.0, total_norm=buf[53])
    # an AdamW run has read its scalars before it writes
    adamw = optim.AdamWPlan([buf[60:64]], [buf[70:74]])
    adamw.run(buf[60], grad_scale=buf[70], total_norm=buf[61])


def _host_list(monkeypatch):
    """Lists over host tensors, and -> what the launches were given."""
    calls = []
    to = torch.Tensor.to
    monkeypatch.setattr(torch.Tensor, "to", lambda t, *a, device=None, **k: to(t, *a, **k))
    monkeypatch.setattr(optim, "_one_device", lambda tensors, what: torch.device("cuda", 0))
    monkeypatch.setattr(optim, "_launch", lambda device, entry, what, *args: calls.append((entry, args)))
    monkeypatch.setattr(optim._List, "workspace", lambda self: torch.empty(64, dtype=torch.int64))
    return calls


@pytest.mark.parametrize("count", [3, 40])
def test_a_given_norm_among_the_gradients_is_copied_first(monkeypatch, count):
    """Scaled in place by one workgroup (or by an earlier launch of a long list) while others read it as the norm."""
    calls = _host_list(monkeypatch)
    buf = torch.arange(10.0 * count + 10)
    ps = _params([buf[10 * i:10 * i + 9] for i in range(count)])
    for k in (0, 4, 8, 10 * count - 2):
        slime_amd.clip_grads_with_norm_(ps, 1.0, buf[k])
        assert calls[-1][0] == "wq_grad_clip_list" and calls[-1][1][-3] != buf[k].data_ptr()
    for k in (9, 19, 10 * count - 1, 10 * count):
        slime_amd.clip_grads_with_norm_(ps, 1.0, buf[k])
        assert calls[-1][1][-3] == buf[k].data_ptr()


def test_scalars_without_an_address_are_refused(host_plans):
    """A wrapper (a sharded tensor, say) has address 0, which the kernels take for "not given": the norm of the local part, a scale
    or a learning rate of one."""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls):
            return torch.Tensor._make_wrapper_subclass(cls, (), dtype=torch.float32, device="cpu")

        def to_local(self):
            return None

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError

    wrapped, flipped = Wrapper(), torch._neg_view(torch.ones(()))
    assert wrapped.data_ptr() == 0
    norm, clip, adamw = optim.GradNormPlan(_lists()), optim.GradClipPlan(_lists()), optim.AdamWPlan(_lists(), _lists())
    for bad in (wrapped, flipped, torch.ones(1).to_sparse()):
        for call in (lambda: norm.run(grad_scale=bad), lambda: clip.run(1.0, grad_scale=bad), lambda: clip.run(1.0, total_norm=bad),
                     lambda: adamw.run(bad), lambda: adamw.run(1.0, grad_scale=bad), lambda: adamw.run(1.0, 1.0, total_norm=bad)):
            with pytest.raises(ValueError, match="one float32 value"):
                call()
    for call in (lambda: clip.run(1.0, total_norm=2.0), lambda: adamw.run(1.0, 1.0, total_norm=2.0)):
        with pytest.raises(ValueError, match="total_norm must be one float32 value"):
            call()
    with pytest.raises(TypeError, match="full tensor"):
        slime_amd.clip_grads_with_norm_(_params(_lists()), 1.0, wrapped)
    assert not host_plans
    clip.run(1.0, grad_scale=torch.nn.Parameter(torch.ones(1)), total_norm=torch.ones(1, 1))


def test_tensors_without_memory_are_refused(host_plans):
    """Released storage and wrappers have address 0; the table would send the kernels there."""
    F = _lib.DTYPE_F32
    released = torch.zeros(8)
    released.untyped_storage().resize_(0)
    for row in ([released.data_ptr(), 1024, 8, F], [1024, 0, 8, F], [0, 0, 8, F, 1024, 1024, 1024, 0], [1024, 0, 8, F, 0, 1024, 1024, 0],
                [1024, 0, 8, F, 1024, 0, 1024, 0], [1024, 0, 8, F, 1024, 1024, 0, 0]):
        empty = [1024, 1024, 0, F] if len(row) == 4 else [0, 0, 0, F, 0, 0, 0, 0]
        with pytest.raises(ValueError, match="no memory"):
            optim._item_table(np.array([empty, row], dtype=np.int64), torch.device("cpu"), "x")
    weight = torch.zeros(4, 8, dtype=torch.bfloat16)
    weight.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="no memory"):                    # it would not be written
        optim.AdamWPlan(_lists(1), _lists(1), weights=[weight])
    optim.AdamWPlan(_lists(1, shape=(0, 3)), _lists(1, shape=(0, 3)), weights=_lists(1, torch.bfloat16, (0, 3)))


@pytest.mark.parametrize("clip", [lambda ps: slime_amd.clip_grad_norm_(ps, 1.0),
                                  lambda ps: slime_amd.clip_grads_with_norm_(ps, 1.0, torch.ones(()))])
def test_strided_gradients_that_share_memory_are_refused(monkeypatch, clip):
    """They are scaled by way of copies, which lie apart: their elements counted twice in the norm and were scaled once."""
    calls = _host_list(monkeypatch)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k))
    x, h = torch.randn(6, 8, 10), torch.randn(6, 8, dtype=torch.float32).to(torch.bfloat16)
    crossing = torch.zeros(200).as_strided((3, 4, 2), (50, 7, 3))
    for shared in ([x[:, :3], x[:, :3]], [x, x[:, :3]], [x[:, :3], x], [x[0], x[..., ::2]], [x[:, :3], x[:, 2:5]],
                   [x[..., ::2], x[..., 1::2], x[:, 3:4, 9:]], [x[:, :3].permute(2, 0, 1), x[2:3, 1:2, 4:5]],
                   [h[:, ::2], h.view(torch.float32)[:, 1:3]], [crossing, torch.as_strided(crossing, (4, 5), (30, 2), 8)],
                   [x[i, :, ::2] for i in range(6)] + [x[3, 4:6]]):
        for order in (shared, shared[::-1]):
            with pytest.raises(ValueError, match="share memory"):
                clip(_params(order))
    assert not calls
    apart = [x[:, :3], x[:, 3:8, ::2], x[:, 3:8, 1::2].permute(1, 2, 0)]
    for fine in (apart, apart[::-1], [x[:, :3], x[:, 3:3], x[:, 3:]], [x[..., ::3], x[..., 1::3], x[..., 2::3]], [h[:, ::2], h[:, 1::2]],
                 [h[:, :2].T, h.view(torch.float32)[:, 1:3]], [x[i, :, j::4] for i in range(6) for j in range(4)],
                 [x[1, 2, 3:5], x[1:, 3:], x[0]]):
        before = [t.clone() for t in fine]
        clip(_params(fine))
        assert all(torch.equal(a, b) for a, b in zip(fine, before))      # nothing was launched: the copies come back as they were
    assert calls
    y = torch.zeros(64 * 9).view(9, 64)
    assert not optim._share_memory([y[:, i] for i in range(64)])
    assert optim._share_memory([y[:, i] for i in range(64)] + [y[4:5, 63:]])


def test_shared_elements_against_a_count():
    """Random pairs of strided views against the sets of their addresses."""
    import random

    rng = random.Random(5)
    buf = torch.zeros(4000)
    seen = set()

    def view():
        dims, reach, shape, stride = rng.randint(1, 3), 0, [], []
        for _ in range(dims):
            shape.append(rng.randint(1, 5))
            stride.append(reach + rng.randint(1, 9))
            reach += stride[-1] * (shape[-1] - 1)
        order = rng.sample(range(dims), dims)
        return buf.as_strided([shape[i] for i in order], [stride[i] for i in order], rng.randint(0, 60))

    index = torch.arange(4000)
    for _ in range(1500):
        a, b = view(), view()
        at = [set(index.as_strided(v.shape, v.stride(), v.storage_offset()).flatten().tolist()) for v in (a, b)]
        shared = bool(at[0] & at[1])
        assert optim._share_memory([a, b]) == shared
        seen.add(shared)
    assert seen == {True, False}


def test_numbers_that_fp32_cannot_hold_are_refused(host_plans):
    """Finite in 64 bits and infinite (or an eps of 0) in the kernels: every gradient or weight became infinite or NaN."""
    clip, adamw = optim.GradClipPlan(_lists()), optim.AdamWPlan(_lists(), _lists())
    most = float(np.finfo(np.float32).max)
    for call in (lambda: clip.run(1.0, grad_scale=1e39), lambda: adamw.run(1e-3, grad_scale=3.5e38), lambda: adamw.run(1e39),
                 lambda: optim.GradNormPlan(_lists()).run(1e300), lambda: optim.AdamWPlan(_lists(), _lists(), weight_decay=1e39),
                 lambda: optim.AdamWPlan(_lists(), _lists(), lr_scale=[1.0, 1e39, 1.0])):
        with pytest.raises(ValueError, match="finite .*in fp32"):
            call()
    for eps in (1e-50, 2.0 ** -150, 5e-324):
        with pytest.raises(ValueError, match="eps"):
            optim.AdamWPlan(_lists(), _lists(), eps=eps)
        assert _lib.load().wq_adamw_items(P, 1, _hyper(eps=eps), P, None) == S
    assert not host_plans
    clip.run(1e39, grad_scale=most)                       # a limit above everything is no limit
    optim.AdamWPlan(_lists(), _lists(), eps=1e-45).run(most)
    optim.AdamWPlan(_lists(), _lists(), eps=0.0, weight_decay=most, lr_scale=most)
    assert _lib.load().wq_adamw_items(None, 1, _hyper(eps=1e-45), P, None) == N_


# ---- norms over ranks ---------------------------------------------------------------------------------------------------------
RANK_NORMS = [(3.0, 4.0), (1e25, 3e25), (1e-30, 2e-30), (0.0, 0.0), (math.inf, 1.0), (1.0, math.nan), (math.nan, math.inf), (3e38, 3e38)]


def _reduce_on_rank(rank, port, results):
    import torch.distributed as dist

    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    for i, norms in enumerate(RANK_NORMS):
        norm = torch.tensor(norms[rank])                 # as a plan on this rank returns it
        total = norm.double().square()
        dist.all_reduce(total)
        results[i, rank, 0] = total.sqrt().float()
        dist.all_reduce(norm.view(torch.int32), op=dist.ReduceOp.MAX)
        results[i, rank, 1] = norm
    dist.destroy_process_group()


def test_norms_over_ranks():
    """The two reductions that the module gives, over two processes."""
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    results = torch.zeros(len(RANK_NORMS), 2, 2).share_memory_()
    torch.multiprocessing.spawn(_reduce_on_rank, (port, results), nprocs=2)
    for (a, b), got in zip(RANK_NORMS, results):
        a, b = (float(torch.tensor(x)) for x in (a, b))
        nan = math.isnan(a) or math.isnan(b)
        two = math.nan if nan else math.inf if math.inf in (a, b) else math.hypot(a, b)
        want = torch.tensor([two, math.nan if nan else max(a, b)], dtype=torch.float64).float()
        assert all(torch.equal(g.nan_to_num(-1.0, posinf=math.inf), want.nan_to_num(-1.0, posinf=math.inf)) for g in got), (a, b, got, want)


def test_updates_refuse_gradients_that_moved(host_plans):
    """zero_grad() drops the gradients by default: the plan kept the old ones and stepped on them without an error."""
    ps = _params(_lists())
    plan = optim.AdamWPlan(ps, [p.grad for p in ps])
    views = optim.AdamWPlan(ps, [p.grad.detach() for p in ps])
    apart = optim.AdamWPlan(ps, _lists())
    plan.run(0.1), views.run(0.1), apart.run(0.1)
    opt = torch.optim.SGD(ps, lr=0.0)
    opt.zero_grad(set_to_none=False)
    sum((p * 2).sum() for p in ps).backward()               # accumulates in place
    plan.run(0.1), views.run(0.1), apart.run(0.1)
    opt.zero_grad()
    plan.run(0.1), views.run(0.1), apart.run(0.1)           # no gradient of its own: whoever drops it may fill the plan's
    assert len(host_plans) == 9
    sum((p * 2).sum() for p in ps[1:]).backward()
    for p in (plan, views):
        with pytest.raises(RuntimeError, match="another gradient tensor"):
            p.run(0.1)
    apart.run(0.1)
    assert len(host_plans) == 10
    fresh = optim.AdamWPlan(ps[1:], [p.grad for p in ps[1:]])
    fresh.run(0.1)
    table = torch.nn.Parameter(torch.zeros(4, 8))
    table.grad = torch.zeros(4, 8).to_sparse()              # its dense sum is elsewhere
    optim.AdamWPlan([table], [torch.zeros(4, 8)]).run(0.1)
    y = torch.zeros(4, requires_grad=True) * 1.0            # not a leaf: has no gradient to compare with, and no warning
    optim.AdamWPlan([y], [torch.zeros(4)]).run(0.1)
    assert len(host_plans) == 13
    ps[0].grad = torch.zeros(4, 8).to_sparse()
    with pytest.raises(RuntimeError, match="another gradient tensor"):
        plan.run(0.1)
