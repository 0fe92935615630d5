"""The plain forms of perf/more_operators.py: passes on the same inputs give the same
outputs and leave the inputs as they were."""

import importlib.util
import random
from pathlib import Path

import pytest
import torch

FILE = Path(__file__).resolve().parents[1] / "perf" / "more_operators.py"


@pytest.fixture(scope="module")
def workloads():
    spec = importlib.util.spec_from_file_location("more_operators", FILE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def tensors(s):
    return {n: v for n, v in s.items() if isinstance(v, torch.Tensor)}


def passes_agree(workloads, s):
    kept = {n: v.detach().clone() for n, v in tensors(s).items()}
    first = {n: v.clone() for n, v in workloads.run(s).items()}
    for n, v in workloads.run(s).items():
        assert torch.equal(v, first[n]), n
    for n, v in tensors(s).items():
        assert torch.equal(v.detach(), kept[n]), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay", [True, False])
def test_a_training_step_keeps_its_inputs(workloads, dtype, decay):
    gen = torch.Generator().manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=gen)
    b, t, c = 2, 70, 5
    s = dict(op="recur train", x=normal(b, t, c).to(dtype), gate=normal(b, t, c).to(dtype),
             input_gate=normal(b, t, c).to(dtype), state=normal(b, c), lengths=None,
             log_decay=-torch.rand(c, generator=gen) if decay else None, want_state=True,
             d_out=normal(b, t, c).to(dtype), d_state=normal(b, c))
    passes_agree(workloads, s)


@pytest.mark.gpu
def test_drawn_cases_keep_their_inputs(workloads):
    """(Single tokens update their states, as they should.)"""
    rng = random.Random(0)
    seen = 0
    while seen < 40:
        case = workloads.draw(rng)
        size = case["c"] * case.get("rows", case.get("b", 1) * case.get("t", 1))
        if case["op"].endswith("step") or size > 1 << 21:
            continue
        seen += 1
        passes_agree(workloads, workloads.prepare(case, seen))
