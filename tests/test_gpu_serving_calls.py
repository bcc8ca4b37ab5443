"""Calls of a serving step's operators on the GPU that their documentation
allows and that differ from an ordinary step's in how the operands lie, how
large they are or which stream they come from; every comparison is for equality."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref
from conftest import case
from test_gpu_serving import (adapter_inputs, attention_inputs, dirty, exp_lut, gpu, rng, run_adapters, run_attention,  # noqa: F401
                              same, verify_inputs, want_adapters)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix", [70, 700])
def test_tails_that_all_slots_share(backend, exp_lut, prefix):
    """A slot stride of 0: every sequence continues with the same tail."""
    case(f"attention shared tail prefix={prefix}")
    s = attention_inputs(81, 6, 2, prefix, 30, 14, 2, 64)
    s["kt"][:], s["vt"][:] = s["kt"][:1], s["vt"][:1]
    d = dict(s, kt=gpu(s["kt"][:1]).expand(s["kt"].shape), vt=gpu(s["vt"][:1]).expand(s["vt"].shape))
    same(run_attention(backend, d, exp_lut), ref.attention(**s, lut=exp_lut), "shared tail")
