"""``FusedAdamW`` and ``clip_gradients`` on the GPU against the oracle: moments
equal float32 arithmetic bit for bit, parameters within the derived bound of the
step in 64 bits, 8-bit codes equal the form written from real arithmetic."""
import math

import numpy as np
import pytest
import torch

from mlx_gsplat_b200 import (_lib, FusedAdamW, FusedMLXAdam, PointerStableChunkedAllocator, clip_gradients,
                             frustum_culling_mlx, rasterize_gaussians_mlx, synthetic)
from mlx_gsplat_b200.adamw import _ENTRY, BLOCK, _clip_entries
from oracle import adamw as oadamw

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}  # a rounding to nearest, relative
TINY = {F32: 0.0, BF16: 2.0 ** -134, F16: 2.0 ** -25}     # and below the normal range
SIZES = [1, 7, 8, 9, 255, 256, 257, 0, 2047, 2048, 2049, 5003]


@pytest.fixture(params=[True, False], ids=["native", "python"])
def reader(request, monkeypatch):
    """The tensors' metadata read natively, or by the checks in Python."""
    if not request.param:
        monkeypatch.setattr(_lib, "tensors", lambda: None)
    else:
        assert _lib.tensors() is not None
    return request.param


def tensors(seed, shapes, dtype, scale=1.0, sparse=0.0):
    gen = torch.Generator().manual_seed(seed)
    out = {}
    for k, s in shapes.items():
        x = torch.randn(s, generator=gen) * torch.exp(2 * torch.randn(s, generator=gen)) * scale
        x = torch.where(torch.rand(s, generator=gen) < sparse, 0.0, x)
        out[k] = x.to(dtype).to(DEV)
    return out


def flat(t):
    return t.detach().float().reshape(-1).cpu().numpy()


def finite(t):
    x = flat(t)
    return np.where(np.isfinite(x), x, np.nan)


class Reference:
    """The oracle's state of one optimizer; ``step`` checks the optimizer against it."""

    def __init__(self, opt, params):
        self.opt, self.params = opt, params
        self.p = {k: flat(p) for k, p in params.items()}
        self.m, self.v = ({k: np.zeros(p.size, np.float32) for k, p in self.p.items()} for _ in range(2))
        self.t = 0

    def check(self, grads, lr=1e-3, decay=None, lr_scales=None, scale=1.0, master=False):
        o = self.opt
        self.t += 1
        got_m, got_v = o.moments()
        for k, g in grads.items():
            gg = flat(g)
            args = dict(beta1=o.beta1, beta2=o.beta2, scale=scale)
            wd = o.weight_decay if decay is None else decay[k]
            pn, _, _, bound = oadamw.step64(self.p[k], gg, self.m[k], self.v[k], lr=lr * (lr_scales or {}).get(k, 1.0),
                                            eps=o.eps, decay=wd, t=self.t, **args)
            self.m[k], self.v[k] = oadamw.step32(gg, self.m[k], self.v[k], **args)
            if o.state_bits == 8:
                self.m[k] = oadamw.values(*oadamw.quantize(self.m[k], self.t, False), False)[:gg.size]
                self.v[k] = oadamw.values(*oadamw.quantize(self.v[k], self.t, True), True)[:gg.size]
            np.testing.assert_array_equal(flat(got_m[k]), self.m[k], err_msg=f"m of {k}")
            np.testing.assert_array_equal(flat(got_v[k]), self.v[k], err_msg=f"v of {k}")
            p = self.params[k]
            held = flat(o._views(o.master_slab)[k]) if master else flat(p)
            dt = F32 if master else p.dtype
            tol = bound + HALF_STEP[dt] * np.abs(pn) + TINY[dt]
            err = np.abs(held - pn)
            assert (err <= tol).all(), (k, (err / np.maximum(tol, 1e-300)).max())
            if master:
                np.testing.assert_array_equal(flat(p), flat(torch.from_numpy(held).to(p.dtype)))
            self.p[k] = held
        assert o.t == self.t
        # padding behind every tensor stays zero
        for slab in o.moment_slabs():
            total = sum(float(x.double().abs().sum()) for x in o._views(slab).values())
            assert abs(float(slab.double().abs().sum()) - total) <= 1e-9 * total


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype,gtype,master", [(F32, F32, False), (F32, BF16, False), (BF16, BF16, False),
                                                (F16, F16, False), (BF16, F32, False), (BF16, BF16, True),
                                                (F16, F16, True)])
def test_step_matches_oracle(bits, ptype, gtype, master):
    shapes = {f"x{i}": (n,) for i, n in enumerate(SIZES)}
    params = tensors(1, shapes, ptype)
    lr_scales, decays = {"x0": 3.0, "x5": 0.0, "x11": 0.05}, {"x3": 0.0, "x8": 2.0}
    opt = FusedAdamW(params, lr=1e-2, weight_decay=0.1, lr_scales=lr_scales, decay_scales=decays, state_bits=bits,
                     master_weights=master)
    ref = Reference(opt, params)
    for s in range(4):
        grads = tensors(10 + s, shapes, gtype, scale=1e-2, sparse=0.3)
        assert opt.step(grads) is None
        ref.check(grads, lr=1e-2, decay={k: 0.1 * decays.get(k, 1.0) for k in shapes}, lr_scales=lr_scales,
                  master=master)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("scale,betas,eps", [(1e-24, (0.9, 0.999), 1e-8), (1e-12, (0.9, 0.999), 1e-15),
                                             (1e15, (0.9, 0.999), 1e-8), (1.0, (0.0, 0.0), 1e-8),
                                             (1.0, (0.0, 0.99), 1e-3), (1.0, (0.95, 0.0), 1e-8)])
def test_gradient_sizes_and_betas(bits, scale, betas, eps):
    """Squares past float32's normal range on both sides, and corrections of betas
    of 0.  (A root of a float32 v that underflows is off by 2^-74 at most, against
    an eps of 1e-8 nothing.)"""
    shapes = {"a": (5000,), "b": (300,)}
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, lr=1e-2, betas=betas, eps=eps, state_bits=bits, weight_decay=0.3)
    ref = Reference(opt, params)
    for s in range(3):
        grads = tensors(10 + s, shapes, F32, scale=scale)
        opt.step(grads)
        ref.check(grads, lr=1e-2)


def test_mixed_types_in_one_step_and_grad_scale(reader):
    shapes = {"a": (33, 5), "b": (2050,), "c": (7, 11, 13), "d": ()}
    params = {**tensors(1, {"a": shapes["a"], "d": ()}, F32), **tensors(2, {"b": shapes["b"]}, BF16),
              **tensors(3, {"c": shapes["c"]}, F16)}
    params = {k: params[k] for k in shapes}
    opt = FusedAdamW(params, lr=1e-2, state_bits=8)
    ref = Reference(opt, params)
    for s in range(3):
        grads = {k: tensors(20 + s, {k: shapes[k]}, dt, scale=50.0)[k]
                 for k, dt in zip(shapes, (BF16, F16, F32, F32))}
        opt.step(grads, grad_scale=1 / 64)
        ref.check(grads, lr=1e-2, scale=1 / 64)


@pytest.mark.parametrize("bits", [32, 8])
def test_strided_rows_leave_their_surroundings(bits, reader):
    """Columns of one slab (a pool's views), an offset view and strided gradients."""
    slab = torch.randn(301, 20, device=DEV)
    back = torch.randn(4000, device=DEV)
    params = {"q": slab[:, 0:4], "m": slab[:, 4:7], "o": slab[:, 7:8], "s": slab[2:250:2, 9:12], "odd": back[3:3000]}
    before, before_back = slab.clone(), back.clone()
    opt = FusedAdamW(params, lr=1e-2, state_bits=bits)
    ref = Reference(opt, params)
    gs = torch.randn(301, 24, device=DEV) * 0.01
    for s in range(3):
        gs = gs.roll(1, 0) * 1.5
        wide = torch.randn(2997, 3, device=DEV)
        grads = {"q": gs[:, 2:6], "m": gs[:, 6:9].contiguous(), "o": gs[:, 9:10], "s": gs[:124, 1:4].t().contiguous().t(),
                 "odd": wide[:, 1] if s else wide[:, 1].contiguous()}
        opt.step(grads)
        ref.check(grads, lr=1e-2)
    np.testing.assert_array_equal(slab[:, 12:].cpu(), before[:, 12:].cpu())
    np.testing.assert_array_equal(slab[:, 8].cpu(), before[:, 8].cpu())
    np.testing.assert_array_equal(slab[1::2, 9:12].cpu(), before[1::2, 9:12].cpu())
    np.testing.assert_array_equal(slab[250:, 9:12].cpu(), before[250:, 9:12].cpu())
    np.testing.assert_array_equal(back[:3].cpu(), before_back[:3].cpu())
    np.testing.assert_array_equal(back[3000:].cpu(), before_back[3000:].cpu())


@pytest.mark.parametrize("bits", [32, 8])
def test_broadcast_gradients_and_missing_ones(bits, reader):
    shapes = {"a": (300,), "b": (40, 9), "c": (3,)}
    params = {k: p.requires_grad_(True) for k, p in tensors(1, shapes, F32).items()}
    opt = FusedAdamW(params, state_bits=bits)
    ref = Reference(opt, params)
    grads = {"a": torch.full((1,), 0.25, device=DEV).expand(300), "b": torch.randn(9, 40, device=DEV).t()}
    opt.step(grads)
    ref.check(grads)
    before = params["b"]._version
    params["b"].grad = torch.randn(40, 9, device=DEV)
    a0 = params["a"].detach().clone()
    opt.step()  # from .grad; a and c have none
    ref.check({"b": params["b"].grad})
    assert params["b"]._version > before and torch.equal(params["a"], a0)
    params["b"].grad = None
    assert opt.step() is None and opt.t == 2  # nothing to do


@pytest.mark.parametrize("count", [25, 368, 369, 900])
def test_more_tensors_than_a_table(count, reader):
    rng = np.random.default_rng(count)
    shapes = {f"x{i}": (int(n),) for i, n in enumerate(rng.integers(0, 700, count))}
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, state_bits=8, max_norm=0.5)
    ref = Reference(opt, params)
    for s in range(2):
        grads = tensors(5 + s, shapes, F32, scale=1e-3)
        norm = opt.step(grads)
        exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
        assert abs(float(norm) - exact) <= 2.0 ** -24 * 1.01 * exact
        ref.check(grads, scale=min(1.0, 0.5 / exact))


# ---------------------------------------------------------------- norm and clipping
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [1e-12, 1.0, 0.25, 1e12])
def test_clip_gradients(dtype, scale, reader):
    if dtype == F16 and scale != 1.0:
        scale = {1e-12: 1e-3, 0.25: 0.25, 1e12: 30.0}[scale]
    shapes = {f"x{i}": (n,) for i, n in enumerate(SIZES + [100_001])}
    grads = tensors(3, shapes, dtype, scale=scale, sparse=0.2)
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    before = {k: g.clone() for k, g in grads.items()}
    # not clipped: the gradients keep their bits
    norm = clip_gradients(grads, exact * 1.01)
    assert norm.dtype == F32 and norm.shape == ()
    if dtype == F16 and scale == 30.0:  # the largest of these pass float16's range: infinities are left
        assert math.isinf(exact) and math.isinf(float(norm))
        clip_gradients(grads, 1.0)
        assert all(torch.equal(grads[k], before[k]) for k in shapes)
        return
    assert abs(float(norm) - exact) <= 2.0 ** -24 * 1.01 * exact
    assert all(torch.equal(grads[k], before[k]) for k in shapes)
    # clipped, into tensors of every type
    for out_type in (F32, BF16, F16) if scale == 1.0 else (dtype,):
        out = {k: torch.full_like(g, 7.0, dtype=out_type) for k, g in grads.items()}
        clip_gradients(grads, 0.3 * exact, out=out)
        for k in shapes:
            want = before[k].double() * 0.3
            # two float32 roundings (factor, product) and the type's
            tol = (HALF_STEP[out_type] + 2.0 ** -23 * 1.01) * want.abs() + TINY[out_type] + 2.0 ** -149
            assert ((out[k].double() - want).abs() <= tol).all(), k
            assert torch.equal(grads[k], before[k])
    # in place, the same bits
    out = {k: torch.empty_like(g) for k, g in grads.items()}
    clip_gradients(list(grads.values()), 0.3 * exact, out=list(out.values()))
    clip_gradients(list(grads.values()), 0.3 * exact)
    assert all(torch.equal(grads[k], out[k]) for k in shapes)


def test_clip_strided_and_repeated_gradients(reader):
    slab = torch.randn(50, 12, device=DEV)
    same = torch.randn(77, device=DEV)
    grads = [slab[:, 1:4], slab[:, 5:6], same, same, torch.randn(6, 50, device=DEV).t()]
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    rows = torch.zeros(77, 4, device=DEV)
    out = [torch.zeros(50, 3, device=DEV), torch.zeros(50, 1, device=DEV), rows[:, 0], torch.zeros(77, device=DEV),
           torch.zeros(50, 6, device=DEV)]
    norm = clip_gradients(grads, 1.0, out=out)
    assert abs(float(norm) - exact) <= 2.0 ** -24 * 1.01 * exact
    for g, o in zip(grads, out):
        want = g.double() / exact
        assert ((o.double() - want).abs() <= 2.0 ** -23 * 1.01 * want.abs()).all()
    assert not rows[:, 1:].any()
    before = slab.clone()
    clip_gradients(grads[:2], 1e-3)
    assert torch.equal(slab[:, 0], before[:, 0]) and torch.equal(slab[:, 4], before[:, 4])
    assert torch.equal(slab[:, 6:], before[:, 6:]) and not torch.equal(slab[:, 1:4], before[:, 1:4])


@pytest.mark.parametrize("count", [24, 25, 500])
def test_clip_more_tensors_than_a_table(count, reader):
    rng = np.random.default_rng(count)
    shapes = {f"x{i}": (int(n),) for i, n in enumerate(rng.integers(0, 5000, count))}
    grads = tensors(3, shapes, F32)
    before = {k: g.clone() for k, g in grads.items()}
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    assert abs(float(clip_gradients(grads, 0.1 * exact)) - exact) <= 2.0 ** -24 * 1.01 * exact
    for k, g in grads.items():
        want = before[k].double() * 0.1
        assert ((g.double() - want).abs() <= 2.0 ** -23 * 1.01 * want.abs()).all(), k


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_not_finite_gradients_are_left(bad):
    g = {"a": torch.randn(5000, device=DEV), "b": torch.zeros(0, device=DEV), "c": torch.randn(3, device=DEV)}
    g["a"][4321] = bad
    before = {k: x.clone() for k, x in g.items()}
    norm = float(clip_gradients(g, 0.1))
    assert not math.isfinite(norm)
    for k in g:
        np.testing.assert_array_equal(g[k].cpu(), before[k].cpu())
    assert float(clip_gradients([torch.zeros(40, device=DEV)], 1.0)) == 0.0
    assert float(clip_gradients([torch.zeros(0, device=DEV)], 1.0)) == 0.0
    huge = torch.full((3000,), 1e37, device=DEV)  # squares past float32, the norm (5.5e38) too
    assert math.isinf(float(clip_gradients([huge], 1.0))) and (huge == 1e37).all()
    huge[400:] = 0.0  # the norm, 2e38, is in range
    assert abs(float(clip_gradients([huge], 1e30)) - 2e38) <= 2.0 ** -23 * 2e38
    # 1e37 itself, the factor and the product are rounded
    assert ((huge[:400].double() - 5e28).abs() <= 3.01 * 2.0 ** -24 * 5e28).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kw", [dict(max_norm=1.0), dict(skip_nonfinite=True)])
def test_step_is_skipped_for_not_finite_gradients(bits, kw):
    shapes = {"a": (700,), "b": (3000,)}
    params = tensors(1, shapes, BF16)
    opt = FusedAdamW(params, state_bits=bits, master_weights=True, **kw)
    opt.step(tensors(2, shapes, BF16))
    state = opt.state_dict()
    before = {k: p.clone() for k, p in params.items()}
    grads = tensors(3, shapes, BF16)
    grads["b"][2999] = math.nan
    assert math.isnan(float(opt.step(grads)))
    after = opt.state_dict()
    assert after["t"] == 1
    for k in ("m", "v", "m_exp", "v_exp", "master"):
        assert torch.equal(after[k], state[k]), k
    assert all(torch.equal(params[k], before[k]) for k in shapes)
    norm = opt.step(tensors(4, shapes, BF16))  # the next step runs
    assert math.isfinite(float(norm)) and opt.t == 2 and not torch.equal(params["a"], before["a"])


def test_skip_alone_does_not_clip():
    shapes = {"a": (700,)}
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, skip_nonfinite=True)
    ref = Reference(opt, params)
    grads = tensors(2, shapes, F32, scale=100.0)
    norm = opt.step(grads, grad_scale=-0.5)
    exact = 0.5 * float(grads["a"].double().norm())
    assert abs(float(norm) - exact) <= 2.0 ** -24 * 1.01 * exact
    ref.check(grads, scale=-0.5)


def test_not_finite_values_stay_in_their_elements():
    shapes = {"a": (1000,), "b": (50,)}
    for bits in (32, 8):
        params = tensors(1, shapes, F32)
        opt = FusedAdamW(params, state_bits=bits)
        grads = tensors(2, shapes, F32)
        grads["a"][300] = math.inf
        opt.step(grads)
        opt.step(tensors(3, shapes, F32))
        bad = ~torch.isfinite(params["a"]).cpu().numpy()
        want = np.zeros(1000, bool)
        if bits == 32:
            want[300] = True
        else:
            want[256:512] = True  # the block's exponent is gone
        np.testing.assert_array_equal(bad, want)
        assert torch.isfinite(params["b"]).all()


# ---------------------------------------------------------------- the 8-bit form
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_load_moments_matches_oracle(dtype, reader):
    shapes = {f"x{i}": (n,) for i, n in enumerate(SIZES)}
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, state_bits=8)
    m = tensors(2, shapes, dtype, sparse=0.2)
    v = {k: x.square() for k, x in tensors(3, shapes, dtype, sparse=0.2).items()}
    if dtype == F32:  # sizes over more than the form's range, in blocks of their own
        m["x11"][256:512] *= torch.exp(8 * torch.randn(256, device=DEV))
        v["x11"][512:768] *= torch.exp(30 * torch.randn(256, device=DEV)).clamp(max=1e30)
        m["x11"][1024:1280] *= 1e-30
        v["x11"][1280:1536] *= 1e-36
        m["x11"][1536:1792] *= 1e30
    opt.load_moments(m, v, t=77)
    assert opt.t == 77
    for dt in (F32, BF16):
        got_m, got_v = opt.moments(dt)
        for k in shapes:
            n = m[k].numel()
            want = oadamw.values(*oadamw.quantize(flat(m[k]), 77, False), False)[:n]
            np.testing.assert_array_equal(finite(got_m[k]), want, err_msg=k)
            want = oadamw.values(*oadamw.quantize(flat(v[k]), 77, True), True)[:n]
            np.testing.assert_array_equal(finite(got_v[k]), want, err_msg=k)
    # what the form holds is kept, at any step
    codes = opt.m.clone(), opt.v.clone(), opt.m_exp.clone(), opt.v_exp.clone()
    opt.load_moments(*opt.moments(), t=1234)
    live = torch.zeros(opt.slab_elements, dtype=torch.bool, device=DEV)
    for view in opt._views(live).values():
        view.fill_(True)
    for a, b, e in zip(codes[:2], (opt.m, opt.v), codes[2:]):
        on = live & (e != 255).repeat_interleave(BLOCK)
        assert torch.equal(a[on], b[on])
    assert torch.equal(codes[2], opt.m_exp) and torch.equal(codes[3], opt.v_exp)


def test_state_dicts():
    shapes = {"a": (700,), "b": (33, 3)}
    grads = [tensors(5 + s, shapes, F32) for s in range(4)]
    runs = []
    for resume in (False, True):
        params = tensors(1, shapes, BF16)
        opt = FusedAdamW(params, state_bits=8, master_weights=True)
        for s, g in enumerate(grads):
            if resume and s == 2:
                d = opt.state_dict()
                opt = FusedAdamW(params, state_bits=8, master_weights=True)
                opt.load_state_dict(d)
            opt.step(g)
        runs.append((params, opt.state_dict()))
    for k in shapes:
        assert torch.equal(runs[0][0][k], runs[1][0][k])
    for k in ("m", "v", "m_exp", "v_exp", "master"):
        assert torch.equal(runs[0][1][k], runs[1][1][k])
    # between the forms: 8 -> 32 -> 8 bits keeps the codes
    wide = FusedAdamW(tensors(1, shapes, BF16), state_bits=32)
    wide.load_state_dict(runs[0][1])
    assert wide.t == 4
    again = FusedAdamW(tensors(1, shapes, BF16), state_bits=8)
    again.load_state_dict(wide.state_dict())
    for a, b in zip(again.moment_slabs(), wide.moment_slabs()):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="other parameters"):
        FusedAdamW(tensors(1, {"a": (700,)}, BF16)).load_state_dict(runs[0][1])


# ---------------------------------------------------------------- streams, graphs, memory
@pytest.mark.parametrize("bits,kw", [(32, {}), (8, dict(max_norm=0.3))])
def test_captured_steps_equal_eager_ones(bits, kw):
    shapes = {"a": (5000,), "b": (33, 3), "c": (1,)}
    grads = [tensors(5 + s, shapes, F32) for s in range(6)]
    lrs = [1e-3 * 0.9 ** s for s in range(6)]
    eager, graphed = tensors(1, shapes, F32), tensors(1, shapes, F32)
    lr = torch.zeros(1, device=DEV)
    a = FusedAdamW(eager, state_bits=bits, lr=lr, **kw)
    for g, x in zip(grads, lrs):
        lr.fill_(x)
        a.step(g)
    lr2 = torch.full((), lrs[0], device=DEV)
    b = FusedAdamW(graphed, state_bits=bits, lr=lr2, **kw)
    static = {k: g.clone() for k, g in grads[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step(static)  # on another stream than the tensors' own
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step(static)
    assert b.t == 1
    for g, x in list(zip(grads, lrs))[1:]:
        for k in shapes:
            static[k].copy_(g[k])
        lr2.fill_(x)
        graph.replay()
    assert a.t == b.t == 6
    assert all(torch.equal(eager[k], graphed[k]) for k in shapes)
    for x, y in zip(a.moment_slabs(), b.moment_slabs()):
        assert torch.equal(x, y)


def test_two_captured_clips_do_not_share_workspace():
    one, two = torch.randn(200_000, device=DEV), torch.randn(300_000, device=DEV)
    outs = torch.empty_like(one), torch.empty_like(two)
    want = [clip_gradients([x], 1.0, out=[torch.empty_like(x)]) for x in (one, two)]
    graphs = []
    for x, o in zip((one, two), outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = clip_gradients([x], 1.0, out=[o])
        graphs.append((g, norm))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, x, o, (_, norm) in zip(want, (one, two), outs, graphs):
        assert torch.equal(w, norm)
        assert abs(float(o.double().norm()) - 1.0) < 1e-6


def test_two_optimizers_on_two_streams():
    shapes = {"a": (70_001,), "b": (333, 3)}
    results = []
    for apart in (False, True):
        params = [tensors(1 + k, shapes, F32) for k in range(2)]
        opts = [FusedAdamW(p, state_bits=8, max_norm=0.1) for p in params]
        grads = [tensors(7 + k, shapes, BF16) for k in range(2)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()] if apart else [torch.cuda.current_stream()] * 2
        torch.cuda.synchronize()
        for _ in range(5):
            for s, o, g in zip(streams, opts, grads):
                with torch.cuda.stream(s):
                    o.step(g)
        torch.cuda.synchronize()
        results.append([x for p, o in zip(params, opts) for x in (*p.values(), o.m, o.v, o.m_exp, o.v_exp)])
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_one_gradient_for_two_parameters_and_changed_settings(reader):
    shapes = {"a": (300,), "b": (300,)}
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, weight_decay=0.0)
    ref = Reference(opt, params)
    g = torch.randn(300, device=DEV)
    opt.step({"a": g, "b": g})
    ref.check({"a": g, "b": g})
    opt.lr, opt.weight_decay, opt.eps, opt.beta1 = 0.03, 0.5, 1e-4, 0.5
    opt.step({"a": g, "b": g})
    # the oracle's correction uses the betas of the step, as the kernel's does
    ref.check({"a": g, "b": g}, lr=0.03)
    with pytest.raises(ValueError):
        opt.weight_decay = -1.0
    opt.beta2 = 1.0
    with pytest.raises(RuntimeError, match="betas"):
        opt.step({"a": g, "b": g})


def test_masters_follow_parameters_when_asked():
    params = tensors(1, {"a": (300,)}, BF16)
    opt = FusedAdamW(params, master_weights=True)
    params["a"].mul_(3.0)
    opt.sync_master()
    assert torch.equal(opt._views(opt.master_slab)["a"], params["a"].float())


def test_inference_tensors(reader):
    with torch.inference_mode():
        g, p = torch.ones(100, device=DEV), torch.zeros(100, device=DEV)
        clip_gradients([g], 1.0)
        FusedAdamW({"a": p}, lr=1.0, weight_decay=0.0).step({"a": g})
    # each gradient is 0.1 up to two roundings, and the first step moves by lr (up to 16 roundings and eps)
    assert ((g - 0.1).abs() <= 0.1 * 3 * 2.0 ** -24).all()
    assert ((p + 1.0).abs() <= 20 * 2.0 ** -24 + 1e-7).all()


def test_replaced_parameter_memory(reader):
    params = {"a": torch.randn(100, device=DEV), "b": torch.randn(30, device=DEV)}
    opt = FusedAdamW(params)
    ref = Reference(opt, params)
    params["a"].data = params["a"].data.clone()
    grads = tensors(2, {"a": (100,), "b": (30,)}, F32)
    opt.step(grads)
    ref.check(grads)
    params["a"].data = torch.randn(50, device=DEV)
    with pytest.raises(ValueError):
        opt.step({"b": grads["b"]})


def test_elements_past_32_bits():
    n = (1 << 31) + 4101
    p = torch.zeros(n, dtype=BF16, device=DEV)
    g = torch.zeros(n, dtype=BF16, device=DEV)
    spots = [slice(0, 600), slice((1 << 31) - 300, (1 << 31) + 300), slice(n - 600, n)]
    gen = torch.Generator().manual_seed(0)
    for s in spots:
        p[s] = torch.randn(600, generator=gen).to(BF16).to(DEV)
        g[s] = torch.randn(600, generator=gen).to(BF16).to(DEV)
    p0 = [flat(p[s]) for s in spots]
    opt = FusedAdamW({"p": p}, lr=0.1, state_bits=8, max_norm=1.0)
    norm = float(opt.step({"p": g}))
    exact = math.sqrt(sum(float(g[s].double().square().sum()) for s in spots))
    assert abs(norm - exact) <= 2.0 ** -24 * 1.01 * exact
    m, v = opt.moments(BF16)
    for s, before in zip(spots, p0):
        lo = s.start // BLOCK * BLOCK
        hi = min(n, -(-s.stop // BLOCK) * BLOCK)
        gg, zero = flat(g[lo:hi]), np.zeros(hi - lo, np.float32)
        mm, vv = oadamw.step32(gg, zero, zero, beta1=0.9, beta2=0.999, scale=1.0 / exact)
        np.testing.assert_array_equal(flat(m["p"][lo:hi]), oadamw.values(*oadamw.quantize(mm, 1, False, first=lo), False)[:hi - lo])
        np.testing.assert_array_equal(flat(v["p"][lo:hi]), oadamw.values(*oadamw.quantize(vv, 1, True, first=lo), True)[:hi - lo])
        pn, _, _, bound = oadamw.step64(before, flat(g[s]), np.zeros(600), np.zeros(600), lr=0.1, beta1=0.9, beta2=0.999,
                                        eps=1e-8, decay=0.01, t=1, scale=1.0 / exact)
        assert (np.abs(flat(p[s]) - pn) <= bound + 2.0 ** -8 * np.abs(pn)).all()


@pytest.mark.parametrize("count", [3, 40])
def test_native_reader_takes_dense_tensors_only(count):
    """The native entries of a clip are those of the checks in Python; strided and
    refused calls are left to these."""
    import ctypes

    from test_adamw import clip_cases
    native = _lib.tensors()
    for k, (g, o, dense, _) in enumerate(clip_cases(count, DEV)):
        e, device = np.zeros(count, _ENTRY), (ctypes.c_int * 2)(-1, -1)
        before = sum(x._version for x in o)
        refused = native.gst_clip(list(g), list(o), e.ctypes.data, count, device)
        assert bool(refused) == (not dense), k
        if dense:
            assert list(device) == [0, 1] and sum(x._version for x in o) > before
            want, _ = _clip_entries(range(count), g, o)
            for name in ("param", "grad", "n", "cols", "param_stride", "grad_stride", "param_type", "grad_type"):
                np.testing.assert_array_equal(e[name], want[name], err_msg=f"{k} {name}")
        else:
            assert sum(x._version for x in o) == before
    e, device = np.zeros(1, _ENTRY), (ctypes.c_int * 2)(-1, -1)
    for bad in (torch.zeros(3), torch.zeros(3, device=DEV, dtype=torch.float64), torch.zeros(3, device=DEV).to_sparse(),
                None, 1.0):
        assert native.gst_clip([bad], [bad], e.ctypes.data, 1, device)
        assert native.gst_fill([bad], None, None, [torch.zeros(3, device=DEV)], e.ctypes.data, 1, 0)
    assert native.gst_fill([torch.zeros(4, device=DEV)], None, None, [torch.zeros(3, device=DEV)], e.ctypes.data, 1, 0)
    assert native.gst_fill(None, None, [torch.zeros(3, device=DEV)], [torch.zeros(3, device=DEV)], e.ctypes.data, 1, 0)


# ---------------------------------------------------------------- refusals with device tensors
def test_refusals_on_the_device(reader):
    params = {"a": torch.zeros(8, device=DEV), "b": torch.zeros(3, device=DEV)}
    with pytest.raises(ValueError, match="one device"):
        FusedAdamW({"a": params["a"], "b": torch.zeros(3)})
    with pytest.raises(ValueError, match="lr"):
        FusedAdamW(params, lr=-1.0)
    with pytest.raises(ValueError, match="tensor lr"):
        FusedAdamW(params, lr=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="tensor lr"):
        FusedAdamW(params, lr=torch.zeros(1))
    with pytest.raises(ValueError, match="max_norm"):
        FusedAdamW(params, max_norm=0.0)
    opt = FusedAdamW(params)
    g = {"a": torch.ones(8, device=DEV), "b": torch.ones(3, device=DEV)}
    with pytest.raises(ValueError, match="shape"):
        opt.step({**g, "b": torch.ones(4, device=DEV)})
    with pytest.raises(ValueError, match="float64"):
        opt.step({**g, "b": g["b"].double()})
    with pytest.raises(ValueError, match="must be on"):
        opt.step({**g, "b": torch.ones(3)})
    with pytest.raises(ValueError, match="sparse"):
        opt.step({**g, "b": g["b"].to_sparse()})
    with pytest.raises(ValueError, match="no parameter named"):
        opt.step({"z": g["a"]})
    with pytest.raises(ValueError, match="no parameter named"):
        opt.step({"a": g["a"], "z": g["b"]})
    with pytest.raises(TypeError, match="by name"):
        opt.step(list(g.values()))
    with pytest.raises(ValueError, match="grad_scale"):
        opt.step(g, grad_scale=math.inf)
    with pytest.raises(ValueError, match="exactly"):
        opt.load_moments({"a": g["a"]}, {"a": g["a"]})
    with pytest.raises(ValueError, match="shape"):
        opt.load_moments({**g, "a": g["b"]}, g)
    with pytest.raises(ValueError, match="step count"):
        opt.load_moments(g, g, t=-1)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        FusedAdamW(params, state_bits=8).moments(F16)
    with pytest.raises(ValueError, match="one device"):
        clip_gradients([g["a"], torch.zeros(3)], 1.0)
    assert not params["a"].any() and opt.t == 0


# ---------------------------------------------------------------- as they are used
@pytest.mark.parametrize("bits", [32, 8])
def test_training_a_scene_with_an_exposure_beside_it(bits):
    """Autograd through the rasterizer, slab views of a pool and a small exposure
    tensor in one optimizer, clipped: every step's update is the oracle's for the
    step's own gradients, and the exposure's gradient agrees with differences."""
    wl = synthetic.WORKLOADS["tiny-3k"]
    g = synthetic.make_gaussians(wl, seed=0, n=400)
    views, K = synthetic.make_cameras(wl, seed=2)
    al = PointerStableChunkedAllocator(500, sh_degree=0, device=torch.device(DEV, 0))
    al.set_initial_gaussians(g)
    names = ("means", "quats", "scales", "opacities", "sh0")
    pools = {k: al.physical_pools[k][:400] for k in names}
    leaves = {k: p.detach().requires_grad_(True) for k, p in pools.items()}
    leaves["exposure"] = torch.eye(3, 4, device=DEV).requires_grad_(True)
    opt = FusedAdamW(leaves, lr=1e-2, weight_decay=0.0, max_norm=1e-3, state_bits=bits)
    ref = Reference(opt, leaves)
    target = torch.rand(wl.height, wl.width, 3, device=DEV)

    def loss_of(step):
        vm = views[step]
        args = [leaves[k].contiguous() for k in names]
        ids = frustum_culling_mlx(args[0].detach(), None, None, vm, K, wl.width, wl.height,
                                  opacities=args[3].detach())
        C, _ = rasterize_gaussians_mlx(*args[:4], args[4][ids.long()], vm, K, wl.width, wl.height, ids,
                                       render_width=wl.width, render_height=wl.height)
        C = C.reshape(wl.height, wl.width, 3) @ leaves["exposure"][:, :3].t() + leaves["exposure"][:, 3]
        return (C - target).square().mean()

    for step in range(3):
        for p in leaves.values():
            p.grad = None
        loss_of(step).backward()
        grads = {k: p.grad for k, p in leaves.items()}
        exact = math.sqrt(sum(float(x.double().square().sum()) for x in grads.values()))
        norm = opt.step()
        assert abs(float(norm) - exact) <= 2.0 ** -24 * 1.01 * exact
        ref.check(grads, lr=1e-2, scale=min(1.0, 1e-3 / exact))
    with torch.no_grad():
        e = leaves["exposure"]
        leaves["exposure"].grad = None
    loss_of(0).backward()
    with torch.no_grad():
        for r, c in ((0, 0), (1, 3)):
            x = float(e[r, c])
            h = 1e-2  # the loss is quadratic in the exposure: a central difference has no error of its own
            e[r, c] = x + h
            up = float(loss_of(0).double())
            e[r, c] = x - h
            down = float(loss_of(0).double())
            e[r, c] = x
            # float32 losses of order 1 differ by 2 h |grad|: their own rounding enters over 2 h
            assert abs((up - down) / (2 * h) - float(e.grad[r, c])) <= 16 * 2.0 ** -24 * max(up, down) / (2 * h) + 1e-3 * abs(float(e.grad[r, c]))


def test_beside_the_pooled_adam():
    """Without weight decay the step is the pooled Adam's formula: both move a
    group alike, up to float32 rounding of the step."""
    shapes = {"means": (500, 3)}
    p = tensors(1, shapes, F32)
    q = {k: x.clone() for k, x in p.items()}
    opt, pooled = FusedAdamW(p, lr=1e-2, weight_decay=0.0, eps=1e-15), FusedMLXAdam(lr=1e-2, eps=1e-15)
    m, v = ({k: torch.zeros_like(x) for k, x in q.items()} for _ in range(2))
    for s in range(3):
        g = tensors(7 + s, shapes, F32)
        before = {k: x.clone() for k, x in p.items()}
        opt.step(g)
        q, m, v = pooled.step(q, g, m, v)
        got_m, got_v = opt.moments()
        for k in shapes:
            assert torch.equal(got_m[k], m[k]) and torch.equal(got_v[k], v[k])
            # each side: at most 16 roundings of the step and 2 of the parameter, a step
            tol = (s + 1) * 2.0 ** -24 * (32 * 1e-2 * 8 + 4 * before[k].abs())
            assert ((p[k] - q[k]).abs() <= tol).all()


# ---------------------------------------------------------------- views that read as the negative of their memory
def negated(x, strided):
    """A tensor of x's values that has the negation bit."""
    if strided:
        return torch.view_as_complex(torch.stack([torch.zeros_like(x), -x], -1)).conj().imag
    return torch._neg_view(-x)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_negated_gradients_and_moments(bits, strided, reader):
    shapes = {"a": (700,), "b": (33, 3)}
    plain, other = tensors(1, shapes, F32), tensors(1, shapes, F32)
    one, two = FusedAdamW(plain, state_bits=bits, max_norm=0.1), FusedAdamW(other, state_bits=bits, max_norm=0.1)
    m = tensors(2, shapes, F32)
    v = {k: x.square() for k, x in tensors(3, shapes, F32).items()}
    one.load_moments(m, v, t=5)
    two.load_moments({**m, "a": negated(m["a"], strided)}, v, t=5)
    g = tensors(4, shapes, F32)
    n = {k: negated(x, strided) for k, x in g.items()}
    assert n["a"].is_neg() and torch.equal(n["a"], g["a"])
    one.step(g)
    two.step({"a": n["a"], "b": g["b"]})
    one.step(g)
    two.step(n)
    assert all(torch.equal(plain[k], other[k]) for k in shapes)
    assert torch.equal(one.m, two.m) and torch.equal(one.v, two.v)
    outs = [[torch.zeros_like(x) for x in g.values()] for _ in range(2)]
    norms = [clip_gradients(list(x.values()), 0.1, out=o) for x, o in zip((g, n), outs)]
    assert torch.equal(*norms) and all(torch.equal(x, y) for x, y in zip(*outs))
    with pytest.raises(ValueError, match="negative"):
        clip_gradients(n, 0.1)
    with pytest.raises(ValueError, match="negative"):
        clip_gradients(g, 0.1, out=n)
    with pytest.raises(ValueError, match="negative"):
        FusedAdamW(n)
    two.lr = torch._neg_view(torch.tensor([-0.5], device=DEV))
    with pytest.raises(ValueError, match="negative"):
        two.step(g)


def test_gradients_that_autograd_negates(reader):
    a, b = (torch.randn(50, device=DEV, requires_grad=True) for _ in range(2))
    c = torch.randn(50, dtype=torch.complex64, device=DEV)
    grads = dict(zip("ab", torch.autograd.grad((torch.complex(a, b).conj() + c).abs().sum(), [a, b])))
    assert grads["b"].is_neg()
    params = {"a": a, "b": b}
    opt = FusedAdamW(params)
    ref = Reference(opt, params)
    opt.step(grads)
    ref.check(grads)


# ---------------------------------------------------------------- parameters whose memory is laid out anew
def test_parameters_laid_out_anew_at_their_address(reader):
    """The address alone does not make a parameter the one that was given: another
    layout or type there is refused, and the old form is taken again."""
    params = {"a": torch.nn.Parameter(torch.randn(12, 12, device=DEV)),
              "b": torch.nn.Parameter(torch.randn(30, device=DEV).to(F16))}
    opt = FusedAdamW(params)
    ref = Reference(opt, params)
    grads = tensors(2, {"a": (12, 12), "b": (30,)}, F32)
    first = {k: p.data for k, p in params.items()}
    before = {k: p.detach().clone() for k, p in params.items()}
    for name, other in (("a", first["a"].t()), ("b", first["b"].view(BF16)), ("a", first["a"][:, :4]),
                        ("a", first["a"].view(144)), ("a", first["a"].view(18, 8)), ("b", torch._neg_view(first["b"]))):
        params[name].data = other
        for given in (grads, {name: grads[name]}):
            with pytest.raises(ValueError, match="no longer"):
                opt.step(given)
        params[name].data = first[name]
        assert all(torch.equal(params[k], before[k]) for k in params) and opt.t == 0
    for p, g in zip(params.values(), grads.values()):
        p.grad = g.to(p.dtype)
    params["a"].data = first["a"].t()
    with pytest.raises(ValueError, match="no longer"):
        opt.step()
    params["a"].data = first["a"]
    opt.step()
    ref.check({k: p.grad for k, p in params.items()})
    # a transposition in place is one too
    x = torch.randn(8, 8, device=DEV)
    opt = FusedAdamW({"x": x})
    x.t_()
    with pytest.raises(ValueError, match="no longer"):
        opt.step({"x": torch.ones(8, 8, device=DEV)})


def test_a_copy_made_lazily_is_not_stepped(reader):
    """A parameter that shares its memory with a lazy copy of it gets memory of its own when it is written."""
    p = torch.randn(300, device=DEV)
    before = p.clone()
    opt = FusedAdamW({"p": p}, lr=0.1)
    ref = Reference(opt, {"p": p})
    copy = torch._lazy_clone(p)
    g = tensors(2, {"p": (300,)}, F32)
    opt.step(g)
    ref.check(g, lr=0.1)
    assert torch.equal(copy, before) and not torch.equal(p, before)
    opt.step(g)  # from its new memory
    ref.check(g, lr=0.1)
    assert torch.equal(copy, before)


# ---------------------------------------------------------------- parameters that miss steps
class CountedReference:
    """The definition with a step count for every tensor: a tensor without a
    gradient keeps its values and moments and does not count the step."""

    def __init__(self, opt, params):
        self.opt, self.params = opt, params
        self.p = {k: flat(p) for k, p in params.items()}
        self.m, self.v = ({k: np.zeros(p.size, np.float32) for k, p in self.p.items()} for _ in range(2))
        self.count = dict.fromkeys(params, 0)
        self.t = 0

    def check(self, grads, lr, scale=1.0):
        o = self.opt
        self.t += any(g.numel() for g in grads.values())  # without an element to move a step does nothing
        got_m, got_v = o.moments()
        for k in self.params:
            if k in grads:
                self.count[k] += 1
                gg = flat(grads[k])
                args = dict(beta1=o.beta1, beta2=o.beta2, scale=scale)
                pn, _, _, bound = oadamw.step64(self.p[k], gg, self.m[k], self.v[k], lr=lr, eps=o.eps,
                                                decay=o.weight_decay, t=self.count[k], **args)
                self.m[k], self.v[k] = oadamw.step32(gg, self.m[k], self.v[k], **args)
                if o.state_bits == 8:  # the roundings' offsets are those of the optimizer's steps
                    self.m[k] = oadamw.values(*oadamw.quantize(self.m[k], self.t, False), False)[:gg.size]
                    self.v[k] = oadamw.values(*oadamw.quantize(self.v[k], self.t, True), True)[:gg.size]
                got = flat(self.params[k])
                err = np.abs(got - pn)
                assert (err <= bound).all(), (k, self.t, (err / np.maximum(bound, 1e-300)).max())
                self.p[k] = got
            else:
                np.testing.assert_array_equal(flat(self.params[k]), self.p[k], err_msg=k)
            np.testing.assert_array_equal(flat(got_m[k]), self.m[k], err_msg=f"m of {k}")
            np.testing.assert_array_equal(flat(got_v[k]), self.v[k], err_msg=f"v of {k}")
        assert o.t == self.t


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [4, 40, 400])
def test_missed_steps_are_not_counted(bits, count, reader):
    """Late and rare gradients get the bias corrections of the steps that their
    own tensor took; one tensor spans many blocks, and tables and lists of
    missing tensors are passed."""
    rng = np.random.default_rng(count)
    shapes = {f"x{i}": (int(n),) for i, n in enumerate(rng.integers(1, 700, count))}
    shapes["x1"], shapes["x2"] = (1_300_001,), (0,)
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, lr=1e-2, state_bits=bits)
    ref = CountedReference(opt, params)
    for s in range(5):
        grads = tensors(10 + s, shapes, F32, scale=1e-2)
        if s != 3:  # the fourth step has all of them
            grads = {k: g for i, (k, g) in enumerate(grads.items()) if (i + s) % 3 == 0 or (i == 1 and s == 4)}
        opt.step(grads)
        ref.check(grads, lr=1e-2)


def test_missed_steps_of_very_many_tensors():
    """More tensors in a list than a table's 16-bit places span."""
    n = 70_001
    gen = torch.Generator().manual_seed(0)
    p, g, g2 = (torch.randn(n, generator=gen).to(DEV) for _ in range(3))
    zero = np.zeros(n)
    params = {f"x{i}": x for i, x in enumerate(p.split(1))}
    opt = FusedAdamW(params, lr=0.1)
    ends = [0, n - 1]
    p0 = flat(p)
    opt.step({f"x{i}": g[i:i + 1] for i in ends})
    args = dict(lr=0.1, beta1=0.9, beta2=0.999, eps=1e-8, decay=0.01)
    p1, m1, v1, bound = oadamw.step64(p0, flat(g), zero, zero, t=1, **args)
    got = flat(p)
    assert (np.abs(got - p1) <= bound)[ends].all() and (got == p0)[1:-1].all()
    opt.step({f"x{i}": x for i, x in enumerate(g2.split(1))})
    m, v = (np.zeros(n, np.float32) for _ in range(2))
    mm, vv = oadamw.step32(flat(g), m, v, beta1=0.9, beta2=0.999)
    m[ends], v[ends] = mm[ends], vv[ends]
    late, _, _, bound_late = oadamw.step64(got, flat(g2), m, v, t=1, **args)
    early, _, _, bound_early = oadamw.step64(got, flat(g2), m, v, t=2, **args)
    assert (np.abs(flat(p) - early) <= bound_early)[ends].all()
    assert (np.abs(flat(p) - late) <= bound_late)[1:-1].all()


@pytest.mark.parametrize("kw", [dict(max_norm=0.5), dict(skip_nonfinite=True)])
def test_skipped_steps_are_missed_by_nobody(kw):
    shapes = {"a": (700,), "b": (3000,)}
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, lr=1e-2, **kw)
    ref = CountedReference(opt, params)
    for s in range(4):
        grads = tensors(10 + s, shapes, F32)
        if s < 2:
            del grads["b"]
        exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
        bad = {k: g.clone() for k, g in grads.items()}
        bad["a"][3] = math.nan
        opt.step(bad)
        opt.step(grads)
        ref.check(grads, lr=1e-2, scale=min(1.0, 0.5 / exact) if "max_norm" in kw else 1.0)


def test_missed_steps_in_a_graph_and_in_the_state():
    shapes = {"a": (700,), "b": (3000,), "c": (5,)}
    params = tensors(1, shapes, F32)
    opt = FusedAdamW(params, lr=1e-2)
    ref = CountedReference(opt, params)
    static = {k: g.clone() for k, g in tensors(5, shapes, F32).items()}
    opt.step(static)
    ref.check(static, lr=1e-2)
    # one graph with every gradient, captured before any was missed, and one without b's
    every, some = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(every):
        opt.step(static)
    part = {k: static[k] for k in "ac"}
    with torch.cuda.graph(some):
        opt.step(part)
    for s, graph in enumerate([every, some, some, every, some, every]):
        for k, g in tensors(20 + s, shapes, F32).items():
            static[k].copy_(g)
        graph.replay()
        ref.check(part if graph is some else static, lr=1e-2)
    # resumed, in either form's number of bits
    d = opt.state_dict()
    for bits in (32, 8):
        again = FusedAdamW({k: p.clone() for k, p in params.items()}, lr=1e-2, state_bits=bits)
        again.load_state_dict(d)
        more = CountedReference(again, dict(zip(shapes, again._params)))
        more.t, more.count = ref.t, dict(ref.count)
        more.m, more.v = ({k: flat(x) for k, x in z.items()} for z in again.moments())
        for part in ({"b": static["b"]}, static):
            again.step(part)
            more.check(part, lr=1e-2)
    # a state without the counts, a set count and loaded moments: every tensor took those steps
    old = {k: x for k, x in d.items() if k != "missed"}
    for change in (lambda: again.load_state_dict(old), lambda: setattr(again, "t", 9),
                   lambda: again.load_moments(*again.moments(), t=12)):
        again.step({"a": static["a"]})
        change()
        more = CountedReference(again, dict(zip(shapes, again._params)))
        more.t = again.t
        more.count = dict.fromkeys(shapes, more.t)
        more.m, more.v = ({k: flat(x) for k, x in z.items()} for z in again.moments())
        again.step(static)
        more.check(static, lr=1e-2)
    # moments loaded without a count leave the counts
    again.step({"a": static["a"]})
    again.load_moments(*again.moments())
    more = CountedReference(again, dict(zip(shapes, again._params)))
    more.t = again.t
    more.count = {"a": more.t, "b": more.t - 1, "c": more.t - 1}
    more.m, more.v = ({k: flat(x) for k, x in z.items()} for z in again.moments())
    again.step(static)
    more.check(static, lr=1e-2)


def test_a_gradient_without_memory_is_not_a_missing_one(reader):
    params = {"a": torch.zeros(8, device=DEV), "b": torch.zeros(8, device=DEV)}
    opt = FusedAdamW(params)
    none = torch._efficientzerotensor((8,), device=DEV)
    for grads in ({"a": none, "b": torch.ones(8, device=DEV)}, {"a": none}):
        with pytest.raises(ValueError, match="no memory"):
            opt.step(grads)
    assert opt.t == 0


# ---------------------------------------------------------------- rows and odd addresses in every type
def laid_out(seed, count, dtype, scale=1.0):
    """name -> tensor: columns of a slab, rows at a distance, odd and even offsets, dense and empty tensors; and the
    buffers that they lie in, with a mask of what the tensors cover."""
    gen = torch.Generator().manual_seed(seed)

    def noise(*shape):
        x = torch.randn(shape, generator=gen) * torch.exp(2 * torch.randn(shape, generator=gen)) * scale
        return x.to(dtype).to(DEV)

    out, backs, masks = {}, [], []

    def add(back, *cuts):
        mask = torch.zeros(back.shape, dtype=torch.bool, device=DEV)
        for cut in cuts:
            out[f"x{len(out)}"] = cut(back)
            cut(mask).fill_(True)
        backs.append(back)
        masks.append(mask)

    add(noise(303, 21), lambda b: b[:, 0:4], lambda b: b[:, 4:5], lambda b: b[1::3, 6:19])
    add(noise(2600), lambda b: b[1:2566], lambda b: b[2570:2570])
    add(noise(70, 97), lambda b: b[:, 3:92])  # rows longer than a warp's step
    add(noise(4100), lambda b: b[:2049])
    while len(out) < count:
        n = int(torch.randint(1, 90, (), generator=gen))
        add(noise(8 * n + 16), lambda b: b[3:3 + n], lambda b: b[n + 8:8 * n + 8].view(7, n)[:, :(n + 1) // 2])
    return out, backs, masks


@pytest.mark.parametrize("count", [7, 60])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype,gtype,master", [(F32, BF16, False), (BF16, BF16, False), (F16, F16, False),
                                                (BF16, F32, False), (F16, BF16, True), (BF16, F16, True)])
def test_rows_and_odd_addresses(bits, ptype, gtype, master, count):
    params, backs, masks = laid_out(1, count, ptype)
    before = [b.clone() for b in backs]
    opt = FusedAdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits, master_weights=master)
    ref = Reference(opt, params)
    for s in range(3):
        grads, _, _ = laid_out(10 + s, count, gtype, scale=1e-2)
        shapes_differ = [k for k in params if grads[k].shape != params[k].shape]
        for k in shapes_differ:  # (the small ones' sizes are drawn)
            grads[k] = torch.randn(params[k].numel() + 1, device=DEV).mul(1e-2).to(gtype)[1:].view(params[k].shape)
        if s == 1:  # dense gradients of strided parameters
            grads = {k: g.contiguous() for k, g in grads.items()}
        opt.step(grads)
        ref.check(grads, lr=1e-2, master=master)
    for b, old, mask in zip(backs, before, masks):
        assert torch.equal(b[~mask], old[~mask])


@pytest.mark.parametrize("count", [7, 60])
@pytest.mark.parametrize("gtype,otype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, F16), (F16, BF16)])
def test_clip_rows_and_odd_addresses(gtype, otype, count):
    grads, _, _ = laid_out(3, count, gtype, scale=0.1)
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    strided, backs, masks = laid_out(3, count, otype)  # the same shapes
    before = [b.clone() for b in backs]
    shifted = {k: torch.empty(g.numel() + 1, dtype=otype, device=DEV)[1:].view(g.shape) for k, g in grads.items()}
    for out in (strided, shifted, {k: torch.empty(g.shape, dtype=otype, device=DEV) for k, g in grads.items()}):
        norm = clip_gradients(grads, 0.3 * exact, out=out)
        assert abs(float(norm) - exact) <= 2.0 ** -24 * 1.01 * exact
        for k, g in grads.items():
            want = g.double() * 0.3
            # two float32 roundings (factor, product) and the type's
            tol = (HALF_STEP[otype] + 2.0 ** -23 * 1.01) * want.abs() + TINY[otype] + 2.0 ** -149
            assert ((out[k].double() - want).abs() <= tol).all(), k
    for b, old, mask in zip(backs, before, masks):
        assert torch.equal(b[~mask], old[~mask])
    if gtype == otype:  # in place, the same bits
        again, backs, masks = laid_out(3, count, gtype, scale=0.1)
        before = [b.clone() for b in backs]
        clip_gradients(again, 0.3 * exact)
        assert all(torch.equal(again[k], strided[k]) for k in grads)
        for b, old, mask in zip(backs, before, masks):
            assert torch.equal(b[~mask], old[~mask])


@pytest.mark.parametrize("odd", ["m", "v", "both"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("count", [12, 40])
def test_load_moments_from_odd_addresses(dtype, odd, count, reader):
    sizes = SIZES + [1 + 37 * i for i in range(count - len(SIZES))]
    shapes = {f"x{i}": (n,) for i, n in enumerate(sizes)}
    opt = FusedAdamW(tensors(1, shapes, F32), state_bits=8)

    def shift(x):
        return torch.cat([x.new_zeros(1), x])[1:]

    m = tensors(2, shapes, dtype, sparse=0.2)
    v = {k: x.square() for k, x in tensors(3, shapes, dtype, sparse=0.2).items()}
    if odd != "v":
        m = {k: shift(x) for k, x in m.items()}
    if odd != "m":
        v = {k: shift(x) for k, x in v.items()}
    opt.load_moments(m, v, t=77)
    got_m, got_v = opt.moments()
    for k in shapes:
        n = m[k].numel()
        want = oadamw.values(*oadamw.quantize(flat(m[k]), 77, False), False)[:n]
        np.testing.assert_array_equal(finite(got_m[k]), want, err_msg=k)
        want = oadamw.values(*oadamw.quantize(flat(v[k]), 77, True), True)[:n]
        np.testing.assert_array_equal(finite(got_v[k]), want, err_msg=k)
    live = torch.zeros(opt.slab_elements, dtype=torch.bool, device=DEV)
    for view in opt._views(live).values():
        view.fill_(True)
    assert not opt.m[~live].any() and not opt.v[~live].any()


# ---------------------------------------------------------------- settings and state
def test_grad_scale_beyond_float32(reader):
    """The kernels hold the scale in float32: one that is infinite there is refused."""
    params = tensors(1, {"a": (300,)}, F32)
    before = params["a"].clone()
    g = tensors(2, {"a": (300,)}, F32, scale=1e-30)
    opt = FusedAdamW(params)
    for scale in (1e39, -1e39, 3.5e38):
        with pytest.raises(ValueError, match="grad_scale"):
            opt.step(g, grad_scale=scale)
    assert opt.t == 0 and torch.equal(params["a"], before)
    ref = Reference(opt, params)
    opt.step(g, grad_scale=3e38)
    ref.check(g, scale=3e38)


@pytest.mark.parametrize("bits", [32, 8])
def test_loaded_moments_keep_no_autograd_graph(bits):
    params = tensors(1, {"a": (300,)}, F32)
    opt = FusedAdamW(params, state_bits=bits)
    m = torch.randn(300, device=DEV, requires_grad=True)
    opt.load_moments({"a": m * 2}, {"a": (m * 3).square()}, t=1)
    assert not opt.m.requires_grad and not opt.v.requires_grad
    if bits == 32:
        assert torch.equal(opt.m[:300], (m * 2).detach())
    opt.t = 2
    opt.load_state_dict(opt.state_dict())


def test_parameters_that_miss_a_step_are_not_marked_as_written(reader):
    params = {k: torch.randn(20, device=DEV, requires_grad=True) for k in "abc"}
    opt = FusedAdamW(params)
    versions = {k: p._version for k, p in params.items()}
    opt.step({"a": torch.ones(20, device=DEV), "b": None})
    params["c"].grad = torch.ones(20, device=DEV)
    opt.step()
    assert params["a"]._version > versions["a"] and params["c"]._version > versions["c"]
    assert params["b"]._version == versions["b"] and opt.t == 2
    assert opt.step({}) is None and opt.step({"a": None}) is None and opt.t == 2
    with pytest.raises(ValueError, match="no parameter named"):
        opt.step({"a": torch.ones(20, device=DEV), "z": torch.ones(20, device=DEV)})
    with pytest.raises(ValueError, match="no parameter named"):
        opt.step({"z": None})
    assert opt.t == 2
