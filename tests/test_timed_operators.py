"""The timed serving operators return the same outputs in both of their forms: as many, in the same places, of the same shapes
and types."""
import importlib.util
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture
def timed():
    spec = importlib.util.spec_from_file_location("timed_operators", ROOT / "perf" / "operators.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _layout(outputs):
    return [None if t is None else (t.shape, t.dtype) for t in outputs]


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("mode", ["same", "int8", "e4m3"])
def test_norm_returns_the_same_in_both_forms(timed, pk, monkeypatch, mode, residual):
    """On the host: the call is a stand-in that returns what `add_rms_norm` is documented to return."""
    def stand_in(x, gamma, residual=None, mode=0, out=None, residual_out=None, scales=None, **_):
        return out, scales, x if residual_out is None else residual_out
    monkeypatch.setattr(timed, "_ops", lambda: SimpleNamespace(lib=pk.lib, ops=SimpleNamespace(add_rms_norm=stand_in)))
    x = torch.randn(3, 32, generator=torch.Generator().manual_seed(1)).half()
    state = dict(kind="norm", mode=mode, x=x, gamma=torch.ones(32).half(), residual_in=x if residual else None,
                 residual_out=torch.empty_like(x) if residual else None,
                 out=torch.empty(3, 32, dtype={"same": torch.float16, "int8": torch.int8, "e4m3": torch.uint8}[mode]),
                 scales=None if mode == "same" else torch.empty(3))
    plain = _layout(timed.run(state))
    timed.own = True
    assert _layout(timed.run(state)) == plain
    assert plain[-1] is None or residual


@pytest.mark.gpu
def test_every_kind_returns_the_same_in_both_forms(timed, cuda):
    cases = [c for c in timed.listed() if c["name"] in ("norm_777x2560_int8", "gemv_1x1024x4096", "plan_7_steps", "attention_1x1_over_700")]
    cases += [dict(kind="norm", rows=5, width=96, type=t, mode=m, residual=False) for t in ("f16", "bf16") for m in ("same", "int8", "e4m3")]
    for case in cases:
        layouts = []
        for own in (False, True):
            timed.own = own
            layouts.append(_layout(timed.run(timed.prepare(case, 3))))
        assert layouts[0] == layouts[1] == _layout_of_exact(timed, case, layouts[0]), case


def _layout_of_exact(timed, case, plain):
    """Values in 64 bits stand in the places of the plain form's outputs, with their shapes."""
    outputs = timed.exact(case, 3)
    assert len(outputs) == len(plain)
    for got, want in zip(outputs, plain):
        assert got is None or tuple(got.shape) == tuple(want[0])
    return plain
