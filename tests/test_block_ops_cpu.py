"""The operators around the bf16 / FP8 linears on a machine without a GPU: refusals of the C ABI
and of the torch functions, and the fake kernels' shapes."""
import ctypes

import pytest
import torch

import flashvsr_optimizations_b200 as fvq
from flashvsr_optimizations_b200 import _lib, ops
from helpers import calls_with_a_tangent

BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _rc(name, *args):
    return getattr(_lib.load(), name)(*args)


@pytest.fixture()
def buf():
    raw = ctypes.create_string_buffer(4096 + 32)
    yield (ctypes.addressof(raw) + 31) // 32 * 32


def test_rms_norm_entry_point_checks(buf):
    def rc(x=buf, rows=4, inner=1, outer=64, step=0, d=64, eps=1e-6, res=None, out=None, y=buf, q=None,
           scale=None, w=buf, f32=0):
        return _rc("fvq_rms_norm", x, rows, inner, outer, step, d, w, ctypes.c_float(eps), res, f32, out,
                   y, q, scale, None)
    for bad in (dict(rows=0), dict(rows=(1 << 30) + 1), dict(inner=0), dict(inner=3), dict(d=0),
                dict(d=16385), dict(outer=-1), dict(step=-1), dict(eps=-1.0), dict(eps=float("nan")),
                dict(x=None), dict(y=None), dict(q=buf), dict(y=None, q=buf), dict(scale=buf),
                dict(res=buf), dict(out=buf)):
        assert rc(**bad) == _lib.FVQ_EINVAL, bad
    for bad in (dict(x=buf + 1), dict(y=buf + 1), dict(w=buf + 1), dict(q=buf, scale=buf + 2),
                dict(res=buf + 1, out=buf), dict(res=buf, out=buf + 2, f32=1)):
        assert rc(**bad) == _lib.FVQ_EALIGN, bad


@pytest.mark.parametrize("fp8", [False, True])
def test_product_entry_points_check(buf, fp8):
    def rc(x=buf, sx=buf, m=4, k=64, stride=64, w=buf, sw=buf, n=64, bias=None, act=0, gated=0, res=None,
           y=buf):
        if fp8:
            return _rc("fvq_fp8_scaled_mm_act", x, sx, m, k, stride, w, sw, n, bias, act, gated, res, y, None)
        return _rc("fvq_linear_act", x, m, k, stride, w, n, bias, act, gated, res, y, None)
    for bad in (dict(m=0), dict(m=(1 << 28) + 1), dict(n=0), dict(n=12), dict(n=(1 << 28) + 8), dict(k=0),
                dict(k=68, stride=80), dict(k=1 << 25, stride=1 << 25), dict(stride=48), dict(stride=68),
                dict(act=5), dict(act=-1), dict(x=None), dict(w=None), dict(y=None)):
        assert rc(**bad) == _lib.FVQ_EINVAL, bad
    for bad in (dict(x=buf + 8), dict(w=buf + 8), dict(y=buf + 8), dict(bias=buf + 2), dict(res=buf + 8)):
        assert rc(**bad) == _lib.FVQ_EALIGN, bad
    if fp8:
        assert rc(sx=None) == _lib.FVQ_EINVAL and rc(sw=None) == _lib.FVQ_EINVAL
        assert rc(k=72, stride=80) == _lib.FVQ_EINVAL          # 16 codes are 16 bytes
        assert rc(sw=buf + 4) == _lib.FVQ_EALIGN and rc(sx=buf + 2) == _lib.FVQ_EALIGN
    assert _rc("fvq_set_linear_kernel", 3) == _lib.FVQ_EINVAL
    assert _rc("fvq_set_linear_kernel", -1) == _lib.FVQ_EINVAL
    assert _rc("fvq_set_linear_kernel", 0) == _lib.FVQ_OK


def test_cache_entry_points_check(buf):
    def wr(k=buf, v=buf, tokens=4, heads=2, d=64, ks=128, kh=64, vs=128, vh=64, slots=buf, kc=buf, s=buf,
           num=8):
        return _rc("fvq_fp8_cache_write", k, v, tokens, heads, d, ks, kh, vs, vh, slots, kc, s, buf, buf, num,
                   None)
    for bad in (dict(tokens=0), dict(tokens=(1 << 31) + 1), dict(heads=0), dict(heads=65536), dict(d=0),
                dict(d=68), dict(d=520), dict(ks=4), dict(kh=-8), dict(vs=12), dict(vh=1), dict(k=None),
                dict(v=None), dict(slots=None), dict(kc=None), dict(s=None), dict(num=-1)):
        assert wr(**bad) == _lib.FVQ_EINVAL, bad
    for bad in (dict(k=buf + 8), dict(v=buf + 2), dict(slots=buf + 4), dict(kc=buf + 4), dict(s=buf + 2)):
        assert wr(**bad) == _lib.FVQ_EALIGN, bad

    def rd(pages=4, page=16, heads=2, d=64, table=buf, batch=2, per=2, lens=buf, most=32, k=buf, kc=buf):
        return _rc("fvq_fp8_cache_read", kc, buf, buf, buf, pages, page, heads, d, table, batch, per, lens,
                   most, k, buf, None)
    for bad in (dict(pages=-1), dict(page=0), dict(heads=0), dict(d=4), dict(batch=0), dict(batch=65536),
                dict(per=0), dict(most=0), dict(table=None), dict(lens=None), dict(k=None), dict(kc=None)):
        assert rd(**bad) == _lib.FVQ_EINVAL, bad
    for bad in (dict(table=buf + 2), dict(lens=buf + 2), dict(k=buf + 8), dict(kc=buf + 4)):
        assert rd(**bad) == _lib.FVQ_EALIGN, bad


def test_valid_calls_without_gpu_fail_loudly(buf):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    no_gpu = (_lib.FVQ_ECUDA, _lib.FVQ_EDEVICE)
    assert _rc("fvq_rms_norm", buf, 4, 1, 64, 0, 64, buf, ctypes.c_float(0.0), None, 0, None, buf, None, None,
               None) in no_gpu
    assert _rc("fvq_linear_act", buf, 4, 64, 64, buf, 64, None, 0, 0, None, buf, None) in no_gpu
    assert _rc("fvq_fp8_cache_write", buf, buf, 1, 2, 64, 128, 64, 128, 64, buf, buf, buf, buf, buf, 8,
               None) in no_gpu


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=BF16)
    c, s = torch.zeros(2, 16, 2, 64).to(F8), torch.zeros(2, 16, 2)
    q, sx = x.to(F8), torch.ones(4, 1)
    for call in (lambda: ops.rms_norm(x), lambda: ops.add_rms_norm(x, x), lambda: ops.rms_norm_fp8(x),
                 lambda: ops.add_rms_norm_fp8(x, x), lambda: ops.linear_act(x, x),
                 lambda: ops.fp8_scaled_mm_act(q, sx, q, sx),
                 lambda: ops.fp8_cache_write(x.view(4, 1, 64), x.view(4, 1, 64), torch.zeros(4).long(), c, s,
                                             c, s),
                 lambda: ops.fp8_cache_read(c, s, c, s, torch.zeros(1, 2).int(), torch.zeros(1).int(), 4)):
        with pytest.raises(RuntimeError, match="expected CUDA tensors"):
            call()


def test_fake_kernels_give_shapes_and_types():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 5, 64, dtype=BF16, device="cuda")
        r = torch.empty(3, 5, 64, dtype=F32, device="cuda")
        assert ops.rms_norm(x).shape == x.shape
        y, s = ops.add_rms_norm(x, r)
        assert y.dtype == BF16 and s.dtype == F32 and s.shape == x.shape
        q, scale, s = ops.add_rms_norm_fp8(x, x)
        assert q.dtype == F8 and scale.shape == (3, 5, 1) and scale.dtype == F32 and s.dtype == BF16
        w = torch.empty(96, 64, dtype=BF16, device="cuda")
        assert ops.linear_act(x, w).shape == (3, 5, 96)
        assert ops.linear_act(x, w, act="silu", gated=True).shape == (3, 5, 48)
        wq, ws = torch.empty(96, 64, dtype=F8, device="cuda"), torch.empty(96, 1, device="cuda")
        y = ops.fp8_scaled_mm_act(q, scale, wq, ws, gated=True)
        assert y.shape == (3, 5, 48) and y.dtype == BF16
        c, cs = torch.empty(7, 16, 2, 64, dtype=F8, device="cuda"), torch.empty(7, 16, 2, device="cuda")
        k, v = ops.fp8_cache_read(c, cs, c, cs, torch.empty(3, 4, dtype=torch.int32, device="cuda"),
                                  torch.empty(3, dtype=torch.int32, device="cuda"), 50)
        assert k.shape == v.shape == (3, 50, 2, 64) and k.dtype == BF16


def test_modules_refuse_cpu_weights_and_bad_shapes():
    lin = torch.nn.Linear
    with pytest.raises(RuntimeError):
        fvq.FP8GatedFFN(lin(64, 128), lin(64, 128), lin(128, 64))
    with pytest.raises(ValueError):
        fvq.FP8GatedFFN(lin(64, 128), lin(64, 96), lin(128, 64))
    with pytest.raises(ValueError):
        fvq.FP8GatedFFN(lin(64, 128), lin(64, 128), lin(128, 32))
    with pytest.raises(ValueError):
        fvq.FP8GatedFFN(lin(64, 128), lin(64, 128, bias=False), lin(128, 64))
    with pytest.raises(ValueError):
        fvq.FP8GatedFFN(lin(64, 128), lin(64, 128), lin(128, 64), act="swish")
    with pytest.raises(ValueError):
        fvq.FP8KVCache(4, 16, 2, 68)
    with pytest.raises(ValueError):
        fvq.FP8KVCache(0, 16, 2, 64)
    with pytest.raises(RuntimeError):
        fvq.FP8KVCache(4, 16, 2, 64, device="cpu")


def test_cache_slot_numbers():
    cache = object.__new__(fvq.FP8KVCache)
    cache.k_codes = torch.zeros(9, 16, 1, 8)
    table = torch.tensor([[4, 2], [7, 0]], dtype=torch.int32)
    got = cache.slots(table, torch.tensor([[0, 15, 16, 31], [5, -1, 32, 17]]))   # 32: past its table
    assert got.dtype == torch.int64
    assert got.tolist() == [64, 79, 32, 47, 117, -1, 144, 1]


def test_slots_on_pages_outside_the_store_are_past_it():
    """A page entry that was never filled in is reported by the write, not taken for padding."""
    cache = object.__new__(fvq.FP8KVCache)
    cache.k_codes = torch.empty(6, 16, 1, 8)
    table = torch.tensor([[3, -1, 6]], dtype=torch.int32)
    got = cache.slots(table, torch.tensor([[0, 15, 16, 31, 32, -5]]))
    assert got[:2].tolist() == [48, 63] and got[5] == -1
    assert (got[2:5] >= 6 * 16).all()


def test_forward_mode_tangents_are_refused():
    """The outputs carry no tangent, so it would be dropped without a word."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        for call in calls_with_a_tangent("cpu"):
            with pytest.raises(RuntimeError, match="no gradient formula"):
                call()
    with pytest.raises(RuntimeError, match="no gradient formula"):
        torch.func.jvp(ops.rms_norm, (torch.ones(4, 64),), (torch.ones(4, 64),))


def test_slots_of_a_table_without_pages():
    """Every position is past such a table; nothing is looked up in it (on a GPU that would be a
    device-side assertion)."""
    cache = object.__new__(fvq.FP8KVCache)
    cache.k_codes = torch.empty(6, 16, 1, 8)
    got = cache.slots(torch.empty(2, 0, dtype=torch.int32), torch.tensor([[0, -1, 40], [-3, 15, 1 << 40]]))
    assert got.dtype == torch.int64 and got[1] == -1 and got[3] == -1
    assert (got[[0, 2, 4, 5]] >= 6 * 16).all()
    assert cache.slots(torch.empty(2, 0, dtype=torch.int32), torch.empty(2, 0, dtype=torch.int64)).shape == (0,)


def test_slots_refuse_what_is_no_table_and_positions():
    cache = object.__new__(fvq.FP8KVCache)
    cache.k_codes = torch.empty(6, 16, 1, 8)
    table, at = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 3, dtype=torch.int64)
    assert cache.slots(table.long(), at.int()).tolist() == [0] * 12
    for bad in ((table, at[:1]), (table[:1], at), (table[0], at), (table, at[:, 0]), (table.float(), at),
                (table, at.double()), (table, at.bool())):
        with pytest.raises(ValueError, match="FP8KVCache.slots"):
            cache.slots(*bad)


@pytest.mark.parametrize("why", ["missing", "no library", "another torch"])
def test_without_the_binding_the_registered_operators_serve(why, monkeypatch, tmp_path):
    """One warning, and the calls go on as the registered operators take them."""
    import warnings
    path = tmp_path / "_fvq_torch.so"
    if why == "no library":
        path.write_bytes(b"not a library")
    monkeypatch.setattr(_lib, "BINDING_PATH", _lib.BINDING_PATH if why == "another torch" else path)
    if why == "another torch":
        monkeypatch.setattr(torch, "__version__", "1.0.0")
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(_lib, "_binding_missing", False)
    x = torch.zeros(4, 64, dtype=BF16)
    with pytest.warns(RuntimeWarning, match="_fvq_torch.so cannot be used"):
        with pytest.raises(RuntimeError, match="expected CUDA tensors"):
            ops.rms_norm(x)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(RuntimeError, match="expected CUDA tensors"):
            ops.linear_act(x, x)
    assert _lib.binding() is None
