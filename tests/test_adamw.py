"""``FusedAdamW`` / ``clip_gradients`` on the CPU: refusals, the layout rules,
the C ABI's argument checks, and the 8-bit form's properties (in the oracle)."""
import ctypes
import math
import os
import shutil
import subprocess
import warnings

import numpy as np
import pytest
import torch

from mlx_gsplat_b200 import FusedAdamW, _lib, clip_gradients
from mlx_gsplat_b200.adamw import _ENTRY, _clip_entries, overlapping, rows_of
from oracle import adamw as oadamw

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")


# ---------------------------------------------------------------- layouts
def test_rows_of():
    slab = torch.zeros(10, 60)
    assert rows_of(slab) == (600, 600)
    assert rows_of(slab[:, 4:7]) == (3, 60)
    assert rows_of(slab[:, 7:8]) == (1, 60)
    assert rows_of(slab[3:7]) == (240, 240)
    assert rows_of(slab[::2]) == (60, 120)
    assert rows_of(torch.zeros(4, 5, 6)[:, :, :3]) == (3, 6)
    assert rows_of(torch.zeros(4, 5, 6)[:, :2]) == (12, 30)
    assert rows_of(torch.zeros(4, 5, 6)[:, :2, :3]) is None  # two strides
    assert rows_of(slab.t()) is None
    assert rows_of(torch.zeros(3, 1).expand(3, 4)) is None
    assert rows_of(torch.zeros(())) == (1, 1)
    assert rows_of(torch.zeros(0, 4)) == (1, 1)


def _over(*tensors):
    return overlapping(tensors, [rows_of(t) for t in tensors])


def test_overlap():
    slab = torch.zeros(10, 60)
    assert _over(slab[:, 0:4], slab[:, 4:7], slab[:, 7:8], slab[:, 8:60]) is None
    assert _over(slab[:, 0:5], slab[:, 4:7]) is not None
    assert _over(slab, slab) is not None
    assert _over(slab, slab[:, 3:5]) is not None
    assert _over(slab[:5], slab[5:]) is None
    assert _over(slab[:5, :3], slab[5:, :3], slab[4:6, 4:5]) is None
    flat = torch.zeros(100)
    assert _over(flat[:50], flat[50:]) is None
    assert _over(flat[:51], flat[50:]) is not None
    assert _over(flat, torch.zeros(100), flat[0:0]) is None
    # one pitch, columns that wrap past the row's end
    assert _over(flat[:90].view(9, 10)[:, 8:], flat[9:99].view(9, 10)[:, 0:2]) is not None
    # pitches of which one divides the other; pitches without a common distance
    assert _over(flat.view(10, 10)[:, :2], flat[2:82].view(4, 20)[:, :2]) is None
    assert _over(flat.view(10, 10)[:, :2], flat[11:91].view(4, 20)[:, :2]) is not None
    assert _over(flat.view(10, 10)[:, :2], flat[2:79].view(7, 11)[:, :2]) is not None


# ---------------------------------------------------------------- refusals
@pytest.mark.parametrize("kw,msg", [
    (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=0.0), "eps"),
    (dict(eps=1e-60), "eps"), (dict(eps=math.nan), "eps"), (dict(weight_decay=-1.0), "weight_decay"),
    (dict(state_bits=16), "state_bits"), (dict(lr_scales={"b": 1.0}), "lr_scales"),
    (dict(decay_scales={"a": math.inf}), "decay_scales"),
])
def test_bad_settings(kw, msg):
    with pytest.raises(ValueError, match=msg):
        FusedAdamW({"a": torch.zeros(3)}, **kw)


@pytest.mark.parametrize("params,msg", [
    ({}, "no parameters"),
    ({"a": torch.zeros(3, dtype=torch.float64)}, "float64"),
    ({"a": torch.zeros(3, dtype=torch.int32)}, "int32"),
    ({"a": torch.zeros(3, 4).t()}, "strides"),
    ({"a": torch.zeros(3).to_sparse()}, "sparse"),
    ({"a": torch.zeros(1).expand(4)}, "strides"),
    ({"a": torch.zeros(3)}, "CUDA"),
])
def test_bad_parameters(params, msg):
    with pytest.raises(ValueError, match=msg):
        FusedAdamW(params)


def test_shared_parameters():
    x = torch.zeros(8)
    with pytest.raises(ValueError, match="share memory"):
        FusedAdamW({"a": x, "b": x})
    with pytest.raises(ValueError, match="share memory"):
        FusedAdamW({"a": x[:5], "b": x[4:]})
    with pytest.raises(TypeError):
        FusedAdamW({"a": [1.0]})


def test_bad_clipping():
    g = torch.zeros(8)
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_gradients([g], bad)
    with pytest.raises(ValueError, match="no gradients"):
        clip_gradients({}, 1.0)
    with pytest.raises(ValueError, match="CUDA"):
        clip_gradients([g], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([g, g], 1.0)
    with pytest.raises(ValueError, match="names"):
        clip_gradients({"a": g}, 1.0, out={"b": g})
    with pytest.raises(ValueError, match="shape"):
        clip_gradients({"a": g}, 1.0, out={"a": torch.zeros(7)})
    with pytest.raises(ValueError, match="strides"):
        clip_gradients([torch.zeros(3, 4).t()], 1.0)
    big = torch.zeros(16)
    with pytest.raises(ValueError, match="another gradient"):
        clip_gradients([big[:8]], 1.0, out=[big[4:12]])
    with pytest.raises(ValueError, match="another gradient"):
        clip_gradients([big[:8], big[8:]], 1.0, out=[big[8:], torch.zeros(8)])
    with pytest.raises(ValueError, match="CUDA"):  # its own gradient's memory is fine
        clip_gradients([big[:8]], 1.0, out=[big[:8]])


def clip_cases(count, device):
    """(gradients, outputs, whether dense and apart, whether refused)"""
    back = torch.zeros(100 * count, device=device)
    gl = [back[100 * k:100 * k + 90 + k % 3] for k in range(count)]
    ol = [torch.zeros(g.shape, dtype=torch.bfloat16 if k % 2 else torch.float32, device=device)
          for k, g in enumerate(gl)]
    wide = torch.zeros(2 * gl[-1].numel(), device=device)
    last = gl[-1].numel()
    return [(gl, gl, True, False), (gl, ol, True, False), (gl, list(gl), True, False),
            (gl[:-1] + [gl[0]], ol[:-1] + [ol[-1].new_zeros(gl[0].shape)], True, False),  # read twice
            (gl, ol[:-1] + [wide[::2]], False, False),                                     # strided
            (gl, gl[1:] + gl[:1], False, True),                                            # in others' memory
            (gl, [ol[-1][:gl[0].numel()]] + ol[1:], False, True),                          # written twice
            (gl[:-1] + [gl[0]], gl[:-1] + [gl[0]], False, True),
            (gl, ol[:-1] + [back[50:50 + last]], False, True),                             # part of another gradient
            (gl, ol[:-1] + [wide[:last].view(-1, 1)], False, True),                        # another shape
            (gl[:-1] + [gl[-1].view(torch.bfloat16)[:9]], gl[:-1] + [gl[-1][:9]], False, True)]  # another type


@pytest.mark.parametrize("count", [3, 40])
def test_entries_of_clipping(count):
    for k, (gl, ol, dense, refused) in enumerate(clip_cases(count, "cpu")):
        if refused:
            with pytest.raises(ValueError, match="shape|share|another"):
                _clip_entries(range(count), gl, ol)
            continue
        e, kept = _clip_entries(range(count), gl, ol)
        assert e["grad"].tolist() == [g.data_ptr() for g in kept] and e["param"].tolist() == [o.data_ptr() for o in ol]
        assert e["n"].tolist() == [g.numel() for g in gl]
        if dense:
            for name in ("cols", "param_stride", "grad_stride"):
                assert e[name].tolist() == [g.numel() for g in gl]
        assert e["grad_type"].tolist() == [0] * count
        assert e["param_type"].tolist() == [int(o.dtype == torch.bfloat16) for o in ol]


def test_calls_are_made_on_the_tensors_device(monkeypatch):
    """Launches go to the device that is current: it is switched for a call on
    another one's tensors, and switched back, also after an error."""
    from mlx_gsplat_b200.adamw import _on_device
    now = [0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: now.__setitem__(0, i))
    for index in (0, 3):
        with _on_device(torch.device("cuda", index)):
            assert now == [index]
        assert now == [0]
        with pytest.raises(KeyError):
            with _on_device(torch.device("cuda", index)):
                raise KeyError
        assert now == [0]


# ---------------------------------------------------------------- C ABI checks (no CUDA call is reached)
def _entry(**kw):
    e = np.zeros(1, _ENTRY)
    e["param"], e["grad"], e["n"], e["cols"] = 4096, 8192, 5, 5
    e["param_stride"] = e["grad_stride"] = 5
    for k, v in kw.items():
        e[k] = v
    return e


def _state(bits=32, **kw):
    d = dict(m=1 << 20, v=2 << 20, m_exp=3 << 20, v_exp=4 << 20, master=None, control=5 << 20)
    d.update(kw)
    return _lib.GsAdamWState(d["m"], d["v"], d["m_exp"], d["v_exp"], d["master"], d["control"], bits)


def _settings(**kw):
    d = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, lr_device=None, norm_partials=None,
             num_partials=0, max_norm=math.inf, norm_out=None)
    d.update(kw)
    return _lib.GsAdamWSettings(*d.values())


@built
@pytest.mark.parametrize("entry,state,settings,msg", [
    (dict(n=-1), {}, {}, b"element count"), (dict(cols=0), {}, {}, b"row length"), (dict(state=100), {}, {}, b"256"),
    (dict(param=0), {}, {}, b"null param"), (dict(grad=0), {}, {}, b"null grad"),
    (dict(param_type=3), {}, {}, b"type"), (dict(grad_type=-1), {}, {}, b"type"), (dict(grad=8194), {}, {}, b"misaligned"),
    (dict(param_stride=4), {}, {}, b"stride"), ({}, dict(bits=16), {}, b"32 or 8"), ({}, dict(m=None), {}, b"null"),
    ({}, dict(control=None), {}, b"null"), ({}, dict(bits=8, m_exp=None), {}, b"exponents"),
    ({}, dict(v=(2 << 20) + 4), {}, b"aligned"), ({}, {}, dict(beta1=1.0), b"betas"), ({}, {}, dict(eps=0.0), b"eps"),
    ({}, {}, dict(grad_scale=math.nan), b"grad_scale"), ({}, {}, dict(lr=math.inf), b"lr"),
    ({}, {}, dict(norm_partials=4096, num_partials=1, max_norm=0.0), b"max_norm"),
])
def test_step_refuses(entry, state, settings, msg):
    lib = _lib.load()
    e = _entry(**entry)
    st = lib.gs_adamw_step(e.ctypes.data, 1, _state(**state), _settings(**settings), None)
    assert st == _lib.GS_ERR_INVALID and msg in lib.gs_last_error(), lib.gs_last_error()


@built
def test_other_entries_refuse_and_skip_nothing_to_do():
    lib = _lib.load()
    assert _ENTRY.itemsize == 80 and ctypes.sizeof(_lib.GsAdamWState) == 56 and ctypes.sizeof(_lib.GsAdamWSettings) == 80
    none = _entry(n=0)
    got = ctypes.c_int64(7)
    assert lib.gs_adamw_step(none.ctypes.data, 1, _state(), _settings(), None) == 0
    assert lib.gs_adamw_step(None, 0, _state(), _settings(), None) == 0
    assert lib.gs_adamw_step(None, 1, _state(), _settings(), None) == _lib.GS_ERR_INVALID
    assert lib.gs_adamw_step(none.ctypes.data, 1, None, _settings(), None) == _lib.GS_ERR_INVALID
    assert lib.gs_grad_norm_partials(none.ctypes.data, 1, None, 0, ctypes.byref(got), None) == 0 and got.value == 0
    e = _entry()
    assert lib.gs_grad_norm_partials(e.ctypes.data, 1, None, 0, ctypes.byref(got), None) == _lib.GS_ERR_INVALID
    assert lib.gs_grad_norm_partials(e.ctypes.data, 1, 4096, 8, None, None) == _lib.GS_ERR_INVALID
    assert lib.gs_clip_gradients(e.ctypes.data, 1, 4096, 1, 0.0, None, None) == _lib.GS_ERR_INVALID
    assert lib.gs_clip_gradients(e.ctypes.data, 1, None, 1, 1.0, None, None) == _lib.GS_ERR_INVALID
    assert lib.gs_moments8_quantize(e.ctypes.data, 1, None, 4096, 4096, 4096, 0, None) == _lib.GS_ERR_INVALID
    assert lib.gs_moments8_dequantize(4096, 4096, 4096, 4096, 100, 0, 4096, 4096, None) == _lib.GS_ERR_INVALID
    assert lib.gs_moments8_dequantize(4096, 4096, 4096, 4096, 256, 2, 4096, 4096, None) == _lib.GS_ERR_INVALID
    assert lib.gs_moments8_dequantize(None, None, None, None, 0, 0, None, None, None) == 0


def test_native_reader_leaves_host_tensors_alone():
    native = _lib.tensors()
    if native is None:
        pytest.skip("helper not built")
    e, device, t = np.zeros(1, _ENTRY), (ctypes.c_int * 2)(-1, -1), torch.zeros(3)
    for items in ([t], {"a": t}, None, (t,), [t, t], 3):
        assert native.gst_fill(items, ["a"], [t], [t], e.ctypes.data, 1, 0) == 1
    assert native.gst_clip([t], [t], e.ctypes.data, 1, device) == 1
    assert native.gst_clip([], [], e.ctypes.data, 0, device) == 1
    assert native.gst_params_unmoved([t], e.ctypes.data, 1) == 1 and t._version == 0
    e["param"] = t.data_ptr()
    assert native.gst_params_unmoved([t], e.ctypes.data, 1) == 0 and t._version == 1


# ---------------------------------------------------------------- the 8-bit form
def test_every_code_is_kept():
    """A block of values on the grid is coded back to itself at any step."""
    for positive in (False, True):
        codes = np.arange(256, dtype=np.uint8)
        if not positive:
            codes[128] = 0  # a signed zero is kept as a code, checked apart
        for e in (64, 100, 127, 180, 254):
            x = oadamw.values(codes, np.array([e], np.uint8), positive)
            assert np.isfinite(x).all()
            for t in (0, 1, 12345):
                c, got = oadamw.quantize(x, t, positive)
                assert got[0] == e
                np.testing.assert_array_equal(c, codes)


@pytest.mark.parametrize("positive", [False, True], ids=["m", "v"])
def test_rounding_is_unbiased_over_steps(positive):
    """The mean over N steps of the values a fixed x is rounded to lies within D
    of x in steps of the grid, D = (3 + (1 / ln(golden) + 2 / ln 3) ln N) / N, the
    discrepancy bound of multiples of sqrt(2) (partial quotients at most 2)."""
    rng = np.random.default_rng(3)
    x = np.exp(rng.normal(0, 2, 512)).astype(np.float32)
    x[::256] = 1e3  # keeps the blocks' exponents
    N = 1000
    total = np.zeros(512)
    for t in range(N):
        total += oadamw.values(*oadamw.quantize(x, t, positive), positive)
    d = (3 + (1 / np.log((1 + 5 ** 0.5) / 2) + 2 / np.log(3)) * np.log(N)) / N
    step = np.exp2(np.frexp(x.astype(np.float64))[1] - 4.0)
    err = np.abs(total / N - x)
    # The blocks' top, 1000 = 15.6 steps of 64, is rounded to 960 or to 1024, so the exponent alternates between
    # those of 2^9 and 2^10, and m's lowest whole binade between 2^-5 and 2^-4.  Above it an element's step does
    # not depend on the exponent and the bound holds; below, the step alternates with the top's offset, and what
    # holds is that each rounding is off by less than the coarser step, 2^-4 / 8.
    whole = x >= (0.0 if positive else 2.0 ** -4)
    assert (err <= (d + 2.0 ** -20) * step)[whole].all()
    assert (err[~whole] < 2.0 ** -7).all()


def test_positive_v_stays_positive():
    x = np.full(256, 1e-30, np.float32)
    x[0] = 1.0
    x[5] = 0.0
    for t in range(50):
        c, _ = oadamw.quantize(x, t, True)
        assert c[5] == 0 and (np.delete(c, 5) > 0).all()


# ---------------------------------------------------------------- views that read as the negative of their memory
def memory(address, n):
    return np.ctypeslib.as_array((ctypes.c_float * n).from_address(int(address))).copy()


@pytest.mark.parametrize("strided", [False, True])
def test_negated_gradients_are_resolved(strided):
    """A gradient with the negation bit (autograd makes them behind ``conj``) is
    read by its values, not by its memory's; nothing is written through one."""
    from types import SimpleNamespace
    if strided:
        g = torch.view_as_complex(torch.arange(1.0, 9.0).view(4, 2)).conj().imag
    else:
        g = torch._neg_view(torch.arange(1.0, 5.0))
    assert g.is_neg()
    want = g.clone()
    host = SimpleNamespace(device=SimpleNamespace(index=-1))  # a host tensor's device index
    e, kept = FusedAdamW._with_grads(host, _entry(n=4, cols=4, param_stride=4), ["a"], [g.shape], [g])
    np.testing.assert_array_equal(memory(e["grad"][0], 4), want)
    assert int(e["grad_stride"][0]) == 4 and torch.equal(kept[0], want)
    e, kept = _clip_entries(range(2), [g, want], [torch.zeros(4), torch.zeros(4)])
    np.testing.assert_array_equal(memory(e["grad"][0], 4), want)
    np.testing.assert_array_equal(memory(e["grad"][1], 4), want)
    assert torch.equal(kept[0], want)
    with pytest.raises(ValueError, match="negative"):
        _clip_entries(range(1), [want], [g])
    with pytest.raises(ValueError, match="negative"):
        clip_gradients([g], 1.0)
    with pytest.raises(ValueError, match="negative"):
        FusedAdamW({"a": g})


def test_native_reader_writes_no_lazy_copy():
    """A parameter whose memory a lazy copy still shares gets its own when a step is to write it, and is then reported
    as moved."""
    native = _lib.tensors()
    if native is None:
        pytest.skip("helper not built")
    e, t = np.zeros(1, _ENTRY), torch.arange(3.0)
    e["param"] = t.data_ptr()
    copy = torch._lazy_clone(t)
    assert native.gst_params_unmoved([t], e.ctypes.data, 1) == 1
    assert t.data_ptr() != e["param"][0]
    e["param"] = t.data_ptr()
    assert native.gst_params_unmoved([t], e.ctypes.data, 1) == 0
    t.zero_()
    assert copy.tolist() == [0.0, 1.0, 2.0]


@built
def test_grad_scale_is_a_float32():
    lib, e = _lib.load(), _entry()
    for scale in (1e39, -1e39):
        st = lib.gs_adamw_step(e.ctypes.data, 1, _state(), _settings(grad_scale=scale), None)
        assert st == _lib.GS_ERR_INVALID and b"grad_scale" in lib.gs_last_error()


@built
def test_counted_calls_pass_over_null_gradients():
    lib = _lib.load()
    e, state = _entry(grad=0), _state()
    assert lib.gs_adamw_step(e.ctypes.data, 1, state, _settings(), None) == _lib.GS_ERR_INVALID
    state.counted = 1
    assert lib.gs_adamw_step(e.ctypes.data, 1, state, _settings(), None) == 0  # no gradient: nothing to do
    state.counted = 2
    assert lib.gs_adamw_step(e.ctypes.data, 1, state, _settings(), None) == _lib.GS_ERR_INVALID
    assert b"counted" in lib.gs_last_error()
    got = ctypes.c_int64(7)
    assert lib.gs_grad_norm_partials(e.ctypes.data, 1, 4096, 8, ctypes.byref(got), None) == 0 and got.value == 0
    assert lib.gs_clip_gradients(e.ctypes.data, 1, 4096, 1, 1.0, None, None) == _lib.GS_ERR_INVALID


# ---------------------------------------------------------------- the native reader's library
@pytest.fixture
def undecided(monkeypatch):
    monkeypatch.setattr(_lib, "_TENSORS", None)
    monkeypatch.setattr(_lib, "_TENSORS_DECIDED", False)


def stub_helper(path, abi):
    """A library at ``path`` that says it was compiled against ``abi`` (None: says nothing)."""
    cc = shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    body = "int gst_fill(void) { return 7; }\n"
    if abi is not None:
        body += f'const char* gst_abi(void) {{ return "{abi}"; }}\n'
    subprocess.run([cc, "-shared", "-fPIC", "-x", "c", "-", "-o", str(path)], input=body.encode(), check=True)


@pytest.mark.parametrize("kind", ["another torch", "no version", "no library", "missing"])
def test_unfit_helper_is_left_out(tmp_path, monkeypatch, undecided, kind):
    """A helper of another torch, or one that does not load, is not called: tensors
    are read in Python, and the reason is given once."""
    path = tmp_path / "libgsplat_tensors.so"
    if kind == "another torch":
        stub_helper(path, "torch 1.0, python 3.0")
    elif kind == "no version":
        stub_helper(path, None)
    elif kind == "no library":
        path.write_text("not a library")
    monkeypatch.setattr(_lib, "TENSORS_PATH", str(path))
    with warnings.catch_warnings(record=True) as caught:
        warnings.simplefilter("always")
        assert _lib.tensors() is None and _lib.tensors() is None
    assert len(caught) == (kind != "missing")
    with pytest.raises(ValueError, match="CUDA"):  # and calls run without it
        clip_gradients([torch.zeros(3)], 1.0)


def test_helper_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    from mlx_gsplat_b200 import build
    path = tmp_path / "libgsplat_tensors.so"
    monkeypatch.setattr(build, "TENSORS_LIB", str(path))
    assert build._tensors_stale()
    stub_helper(path, _lib.tensors_abi())
    os.utime(path, (2 ** 33, 2 ** 33))
    assert build._tensors_stale()  # lacks the functions: not a helper that loads
    stub = tmp_path / "other.so"
    stub_helper(stub, "torch 1.0, python 3.0")
    os.utime(stub, (2 ** 33, 2 ** 33))
    monkeypatch.setattr(build, "TENSORS_LIB", str(stub))
    assert build._tensors_stale()
    if _lib.tensors() is not None:
        monkeypatch.setattr(build, "TENSORS_LIB", _lib.TENSORS_PATH)
        monkeypatch.setattr(build, "_older", lambda *a: False)
        assert not build._tensors_stale()


def test_build_does_without_the_helper(tmp_path, monkeypatch, capsys):
    """Where the helper cannot be compiled the build goes on, and an old one is removed."""
    from mlx_gsplat_b200 import build
    path = tmp_path / "libgsplat_tensors.so"
    path.write_text("of other sources")
    monkeypatch.setattr(build, "TENSORS_LIB", str(path))
    monkeypatch.setattr(build, "_stale", lambda *a: False)
    monkeypatch.setenv("CXX", "/bin/false")
    assert build.build() == build.LIB
    assert not path.exists() and "read in Python" in capsys.readouterr().err
    monkeypatch.setenv("CXX", str(tmp_path / "no such compiler"))
    assert build.build() == build.LIB


# ---------------------------------------------------------------- where the 8-bit form ends
@pytest.mark.parametrize("size", [2.0 ** -3, 2.0 ** -20 * 1.3, 2.0 ** -29 * 1.7, 2.0 ** -32 * 1.1, 2.0 ** -33,
                                  2.0 ** -33 * 0.99, 2.0 ** -35, 2.0 ** -60])
def test_v_ends_at_a_step(size):
    """Beside a largest value of 1 the lowest step is 2^-33.  From there up the mean of
    the roundings lies within the discrepancy bound (see above) of the value; what
    is below, and not 0, is held as that step: too large."""
    x = np.full(256, size, np.float32)
    x[0] = 1.0
    n = 1000
    got = np.array([oadamw.values(*oadamw.quantize(x, t, True), True) for t in range(n)], np.float64)
    assert (got[:, 0] == 1.0).all()
    if size < 2.0 ** -33:
        assert (got[:, 1:] == 2.0 ** -33).all()
        return
    d = (3 + (1 / np.log((1 + 5 ** 0.5) / 2) + 2 / np.log(3)) * np.log(n)) / n
    step = max(2.0 ** (math.frexp(size)[1] - 4), 2.0 ** -33)
    assert (np.abs(got[:, 1:].mean(0) - float(np.float32(size))) <= (d + 2.0 ** -20) * step).all()


def test_v_of_small_gradients_stays_at_the_step():
    """Elements whose gradients stay below 2^-16.5 of the block's largest: their v
    is one step, 2^-33 of the block's, however small they are, and with no
    gradient at all it does not return to 0.  (beta2 = 1/2 keeps the largest at
    1; a v of one step and a square below it have a mean below it, which is
    rounded to one step or to 0, and a positive v is never 0.)"""
    g = np.zeros(256, np.float32)
    g[0], g[1:100], g[100:200] = 1.0, 2.0 ** -17, 2.0 ** -30
    v = np.zeros(256, np.float32)
    v[0] = 1.0
    v[200:250] = 2.0 ** -33
    for t in range(200):
        v = oadamw.values(*oadamw.quantize(np.float32(0.5) * v + np.float32(0.5) * (g * g), t, True), True)
        assert v[0] == 1.0 and (v[1:250] == 2.0 ** -33).all() and (v[250:] == 0.0).all()


@pytest.mark.parametrize("positive", [False, True], ids=["m", "v"])
def test_grids_are_nested_downward(positive):
    """Where the block's largest value falls, what the form held is kept exactly; where
    it rises, values below the new lowest whole binade are rounded again, by
    less than the new step, and no others."""
    top = oadamw.V_TOP if positive else oadamw.M_TOP
    codes = np.arange(256, dtype=np.uint8)
    if not positive:
        codes[128:] = 0
    held = oadamw.values(codes, np.array([127], np.uint8), positive)
    held[-1] = 1.0  # the largest of these is below 2, and one at least keeps the exponent
    for t in (0, 5, 77):
        lower = held.copy()
        lower[lower >= 2.0 ** -4] = 0.0
        lower[-1] = 2.0 ** -5  # the exponent falls by five
        c, e = oadamw.quantize(lower, t, positive)
        assert e[0] == 122
        np.testing.assert_array_equal(oadamw.values(c, e, positive), lower)
        higher = held.copy()
        higher[-1] = 4.0  # and rises by two
        c, e = oadamw.quantize(higher, t, positive)
        assert e[0] == 129
        got = oadamw.values(c, e, positive)
        lowest = 2.0 ** (2 - (top - 1))
        np.testing.assert_array_equal(got[higher >= lowest], higher[higher >= lowest])
        assert (np.abs(got - higher) < lowest / 8).all()
        assert (got != higher).any()
