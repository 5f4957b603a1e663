"""Helpers shared by the tests (fixture loading, device transfer, rcp tables)."""
from __future__ import annotations

import json

import numpy as np
import pytest

from conftest import GOLDEN


def golden_meta() -> dict:
    p = GOLDEN / "golden_meta.json"
    if not p.exists():
        pytest.skip("golden fixtures not generated yet (tests/golden/make_golden.py on a B200)")
    return json.loads(p.read_text())


def golden(name: str) -> dict:
    p = GOLDEN / f"{name}.npz"
    if not p.exists():
        pytest.skip(f"golden fixture {name} missing")
    with np.load(p) as z:
        return {k: z[k] for k in z.files}


def table_from(args: np.ndarray, res: np.ndarray) -> dict:
    return dict(zip(np.asarray(args, dtype=np.uint32).tolist(),
                    np.asarray(res, dtype=np.uint32).tolist()))


def f32_from_bits(b) -> np.float32:
    return np.asarray(b, dtype=np.uint32).view(np.float32).reshape(-1)[0]


def bits_to_dev(bits: np.ndarray):
    import torch
    return torch.from_numpy(np.ascontiguousarray(bits).astype(np.int16)).view(torch.bfloat16).cuda()


def dev_to_bits(t) -> np.ndarray:
    import torch
    return t.detach().contiguous().cpu().view(torch.int16).numpy().view(np.uint16)


def gpu_rcp_table(x_bits: np.ndarray, g: float) -> dict:
    """rcp.approx.ftz.f32 measured on the GPU for every argument the oracle needs."""
    import torch
    from oracle import nvfp4_oracle as O
    import flashvsr_optimizations_b200 as fvq
    args = np.array(O.rcp_arguments(x_bits, g), dtype=np.uint32)
    res = fvq.ops.rcp_approx_probe(torch.from_numpy(args.view(np.float32)).cuda())
    return table_from(args, res.cpu().numpy().view(np.uint32))


def calls_with_a_tangent(device: str) -> list:
    """Calls of the block operators, each with one argument that carries a forward-mode tangent
    (make and call them inside a dual level)."""
    import torch
    from torch.autograd.forward_ad import make_dual
    from flashvsr_optimizations_b200 import ops

    def dual(t):
        return make_dual(t, torch.ones_like(t))
    p = torch.ones(8, 64, dtype=torch.bfloat16, device=device)
    s, i = torch.ones(8, 1, device=device), torch.zeros(1, dtype=torch.int32, device=device)
    kv, slots = p.view(8, 1, 64), torch.arange(8, device=device)
    q = p.to(torch.float8_e4m3fn)
    codes, scale = q.view(2, 4, 1, 64), s.view(2, 4, 1)
    x = dual(p)
    return [lambda: ops.rms_norm(x), lambda: ops.rms_norm(p, dual(p[0])), lambda: ops.add_rms_norm(p, x),
            lambda: ops.rms_norm_fp8(x), lambda: ops.add_rms_norm_fp8(x, p), lambda: ops.linear_act(x, p),
            lambda: ops.linear_act(p, x), lambda: ops.linear_act(p, p, residual=dual(torch.ones_like(p[:, :8]))),
            lambda: ops.fp8_scaled_mm_act(q, dual(s), q, s),
            lambda: ops.fp8_cache_write(kv, dual(kv), slots, codes, scale, codes, scale),
            lambda: ops.fp8_cache_read(codes, dual(scale), codes, scale, i.view(1, 1), i, 4)]
