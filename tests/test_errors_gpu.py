"""Failure detection without faulting the GPU: every pipeline wait inside the
GEMM is bounded in wall time.  A wait limit of 1 ns makes the waits give up;
the kernel then drains its own copies and MMAs, frees TMEM, sets the device
error word and returns.  The host reads the word, and the context stays
usable for the next, normal launch."""
import numpy as np
import pytest
import torch

from flashvsr_optimizations_b200 import ops
from oracle import nvfp4_oracle as O

pytestmark = pytest.mark.gpu


def _operands(m, n, k, seed):
    rng = np.random.default_rng(seed)
    def op(rows):
        codes = rng.integers(0, 256, size=(rows, k // 2), dtype=np.uint8)
        sf = np.zeros(O.sf_swizzled_size(rows, k), dtype=np.uint8)
        sf[O.sf_swizzled_offsets(rows, k // 16)] = rng.integers(0x30, 0x40, size=(rows, k // 16),
                                                                 dtype=np.uint8)
        return torch.from_numpy(codes).cuda(), torch.from_numpy(sf).cuda()
    return op(m), op(n)


@pytest.mark.parametrize("gelu", [False, True])
def test_wait_timeout_sets_error_word_and_context_survives(gelu):
    (a, asf), (w, wsf) = _operands(512, 1024, 1536, seed=3)
    g = torch.ones(1, device="cuda")
    assert ops.read_device_error() == 0
    ref, _ = ops.nvfp4_gemm(a, asf, g, w, wsf, g, gelu=gelu)
    try:
        ops.set_wait_limit(1)                      # 1 ns: waits give up at once
        ops.nvfp4_gemm(a, asf, g, w, wsf, g, gelu=gelu)
        flags = ops.read_device_error()            # synchronises, returns and clears
    finally:
        ops.set_wait_limit(0)
    assert flags != 0
    assert ops.read_device_error() == 0
    again, _ = ops.nvfp4_gemm(a, asf, g, w, wsf, g, gelu=gelu)
    torch.cuda.synchronize()
    assert torch.equal(again, ref)
    assert ops.read_device_error() == 0


def test_fused_quantizer_grid_wait_timeout_sets_error_word():
    """The fused amax+quantize kernel's grid barrier is bounded as well: with a
    1 ns limit the CTAs that wait give up (kErrWaitGrid, bit 5), the barrier is
    still re-armed by the last CTA to arrive, and the next call is exact."""
    from flashvsr_optimizations_b200 import _lib, workloads as W
    xb = W.gaussian(7680, 1536, seed=21)
    x = torch.from_numpy(xb.astype(np.int16)).view(torch.bfloat16).cuda()
    g_ref = ops.global_scale(x)
    q_ref, s_ref = ops.nvfp4_quantize(x, g_ref)
    lib = _lib.load()
    ws = torch.zeros(lib.fvq_amax_workspace_bytes(), dtype=torch.uint8, device="cuda")
    q, s = torch.empty_like(q_ref), torch.empty_like(s_ref)
    g = torch.empty(1, dtype=torch.float32, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    call = lambda: _lib.call("fvq_nvfp4_quantize_dynamic", x.data_ptr(), 7680, 1536, None,  # noqa: E731
                             g.data_ptr(), q.data_ptr(), s.data_ptr(), ws.data_ptr(), ws.numel(), st)
    assert ops.read_device_error() == 0
    try:
        ops.set_wait_limit(1)
        call()
        flags = ops.read_device_error()
    finally:
        ops.set_wait_limit(0)
    assert flags & (1 << 5), flags
    assert not ws[:4].any(), "the arrival counter is re-armed even after timeouts"
    call()
    torch.cuda.synchronize()
    assert ops.read_device_error() == 0
    assert g.item() == g_ref.item() and torch.equal(q, q_ref) and torch.equal(s, s_ref)


# Waits that run out in the middle of a kernel: from shorter than a first load to longer than the
# whole launch.  Bits 0 to 2 of the error word are waits of the producer, the MMA issuer and the
# epilogue; bit 3, a teardown that did not complete, must not appear, and a result without a bit is
# the result.
LIMITS = [1000, 1500, 2000, 3000, 4000, 6000, 8000, 12000, 16000, 32000, 64000]


def give_up(call, want):
    try:
        for limit in LIMITS:
            ops.set_wait_limit(limit)
            got = call()
            flags = ops.read_device_error()
            assert flags & ~7 == 0, (limit, flags)
            if flags == 0:
                assert torch.equal(got, want), limit
    finally:
        ops.set_wait_limit(0)
    assert torch.equal(call(), want)
    assert ops.read_device_error() == 0


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", [(24, 1536, 8960), (128, 8960, 1536), (16, 64, 64), (100, 264, 16384)])
def test_split_product_gives_up_anywhere(m, n, k, fp8):
    x = torch.randn(m, k, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    w = torch.randn(n, k, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    if fp8:
        args, fn = (*ops.fp8_row_quant(x), *ops.fp8_row_quant(w)), ops.fp8_scaled_mm_act
    else:
        args, fn = (x, w), ops.linear_act
    ops.set_linear_kernel(1)
    try:
        give_up(lambda: fn(*args), fn(*args))
    finally:
        ops.set_linear_kernel(0)


def fp8_rows(m, k, seed):
    x = torch.randn(m, k, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")
    return ops.fp8_row_quant(x.to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", [(512, 1024, 1536), (1000, 1536, 8960)])
@pytest.mark.parametrize("kind", ["nvfp4", "nvfp4_gelu", "fp8"])
def test_one_sm_gemm_gives_up_anywhere(kind, m, n, k):
    if kind == "fp8":
        (a, sa), (w, sw) = fp8_rows(m, k, 1), fp8_rows(n, k, 2)

        def call():
            return ops.fp8_scaled_mm(a, sa, w, sw)
    else:
        (a, asf), (w, wsf) = _operands(m, n, k, seed=3)
        g = torch.ones(1, device="cuda")

        def call():
            return ops.nvfp4_gemm(a, asf, g, w, wsf, g, gelu=kind == "nvfp4_gelu")[0]
    from flashvsr_optimizations_b200 import _lib
    _lib.call("fvq_set_gemm_pairing", 0)
    _lib.call("fvq_set_fp8_gemm_pairing", 0)
    try:
        give_up(call, call())
    finally:
        _lib.call("fvq_set_gemm_pairing", 1)
        _lib.call("fvq_set_fp8_gemm_pairing", 1)


@pytest.mark.parametrize("m,n,k", [(256, 256, 512), (512, 1024, 1536), (1536, 1536, 8960), (7680, 1536, 1536)])
@pytest.mark.parametrize("kind", ["nvfp4", "nvfp4_replicated", "fp8", "bf16_product", "fp8_product", "gated_product"])
def test_pair_gemm_gives_up_anywhere(kind, m, n, k):
    """Either CTA of a pair may give up first, with loads of the other's on the way."""
    from flashvsr_optimizations_b200 import _lib
    if kind == "fp8" or kind == "fp8_product":
        (a, sa), (w, sw) = fp8_rows(m, k, 1), fp8_rows(n, k, 2)
        fn = ops.fp8_scaled_mm if kind == "fp8" else ops.fp8_scaled_mm_act

        def call():
            return fn(a, sa, w, sw)
    elif kind.endswith("product"):
        gated = kind == "gated_product"
        x = torch.randn(m, k, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
        w = torch.randn(n, k, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
        r = torch.randn(m, n // (1 + gated), generator=torch.Generator("cuda").manual_seed(3), device="cuda")

        def call():
            return ops.linear_act(x, w, act="silu", gated=gated, residual=r.to(torch.bfloat16))
    else:
        (a, asf), (w, wsf) = _operands(m, n, k, seed=3)
        g = torch.ones(1, device="cuda")
        lib = _lib.load()
        rep = torch.empty(lib.fvq_w_scales_replicated_bytes(n, k), dtype=torch.uint8, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        _lib.call("fvq_replicate_w_scales", wsf.data_ptr(), n, k, rep.data_ptr(), st)

        def call():
            if kind == "nvfp4":
                return ops.nvfp4_gemm(a, asf, g, w, wsf, g)[0]
            out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
            _lib.call("fvq_nvfp4_gemm_wrep", a.data_ptr(), asf.data_ptr(), g.data_ptr(), w.data_ptr(), rep.data_ptr(),
                      g.data_ptr(), None, out.data_ptr(), m, n, k, st)
            return out
    _lib.call("fvq_set_gemm_pairing", 2 if kind == "nvfp4_replicated" else 1)
    _lib.call("fvq_set_fp8_gemm_pairing", 2)
    ops.set_linear_kernel(2)
    try:
        give_up(call, call())
    finally:
        _lib.call("fvq_set_gemm_pairing", 1)
        _lib.call("fvq_set_fp8_gemm_pairing", 1)
        ops.set_linear_kernel(0)
