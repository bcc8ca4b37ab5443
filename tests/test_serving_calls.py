"""What the calls of a serving step hand to the library, without a GPU: the
library is replaced by a recorder, so that the operands' addresses, strides and
sizes can be held against the memory that the tensors own."""
from __future__ import annotations

import pytest
import torch

from test_serving_host import adapter_args, attention_args, verify_args


class Recorder:
    """Every entry of the library: notes the call, returns success (a workspace function: `nbytes`)."""

    def __init__(self, log, nbytes=256):
        self.log, self.nbytes = log, nbytes

    def __getattr__(self, name):
        def entry(*args):
            self.log.append((name, args))
            return self.nbytes if name.endswith("_workspace") else 0
        return entry


@pytest.fixture
def recorded(monkeypatch):
    """A backend without a context, on CPU tensors, and the list of its calls of the library."""
    from myelith_amd import backend
    b = backend.RocmBackend.__new__(backend.RocmBackend)
    b._h, b._device_id = None, 0
    log = []
    recorder = Recorder(log)
    monkeypatch.setattr(backend, "lib", lambda: recorder)
    monkeypatch.setattr(backend.RocmBackend, "_need_here", lambda *a: None)
    return b, log


def one(t, dim):
    """t's first place of dimension dim, held for all of them: a stride of 0."""
    return t.narrow(dim, 0, 1).expand(t.shape)


# ---- strides of 0 ---------------------------------------------------------------------

def test_expanded_operands_are_refused(recorded):
    """An expanded tensor owns fewer elements than its shape says: taken for a dense one, a
    kernel would read (or write) behind it."""
    b, log = recorded
    ad, at, ve = adapter_args(), attention_args(), verify_args()
    at["out"], ad["out"] = torch.zeros_like(at["q"]), torch.zeros((3, 5), dtype=torch.int16)
    cases = [(b.linear_w8a16_adapters_dev, ad, "x", (0, 1)), (b.linear_w8a16_adapters_dev, ad, "out", (0, 1)),
             (b.attention_prefix_dev, at, "q", (0, 1, 2)), (b.attention_prefix_dev, at, "out", (0, 1, 2)),
             (b.attention_prefix_dev, at, ("k_prefix", "v_prefix"), (0, 1, 2)),
             (b.attention_prefix_dev, at, ("k_tail", "v_tail"), (1, 2, 3)),
             (b.verify_drafts_dev, ve, "target", (0, 1, 2)), (b.verify_drafts_dev, ve, "draft", (0, 1, 2))]
    for call, args, names, dims in cases:
        for dim in dims:
            names = (names,) if isinstance(names, str) else names
            with pytest.raises(ValueError):
                call(**dict(args, **{n: one(args[n], dim) for n in names}))
                pytest.fail(f"{names} expanded in dimension {dim}: {log[-1]}")
    # one row a sequence: the sequences' stride is the rows'
    z = torch.zeros((2, 1, 50), dtype=torch.int32)
    with pytest.raises(ValueError):
        b.verify_drafts_dev(one(z, 0), torch.zeros((2, 0), dtype=torch.int64), torch.zeros((2, 1), dtype=torch.int64),
                            exp_lut=ve["exp_lut"])


def test_tails_that_all_slots_share(recorded):
    """A slot stride of 0 is a place that a kernel can read: it is passed on."""
    b, log = recorded
    a = attention_args()
    b.attention_prefix_dev(**dict(a, k_tail=one(a["k_tail"], 0), v_tail=one(a["v_tail"], 0)))
    name, args = log[-1]
    assert name == "myl_attention_prefix_dev" and args[15:17] == (0, 5 * 64)  # slots, heads apart


def test_dimensions_of_one_element_take_the_dense_stride(recorded):
    """Where a dimension has one element its stride says nothing (torch may leave anything there)."""
    b, log = recorded
    odd = lambda dtype, shape, strides: torch.zeros(4096, dtype=dtype).as_strided(shape, strides)
    b.linear_w8a16_adapters_dev(**adapter_args(x=odd(torch.int16, (1, 32), (3, 1)), ids=torch.zeros(1, dtype=torch.int32)))
    assert log[-1][1][3] == 32
    z = lambda *s: torch.zeros(s, dtype=torch.int16)
    b.attention_prefix_dev(**attention_args(q=odd(torch.int16, (1, 1, 64), (0, 0, 1)), k_prefix=odd(torch.int16, (1, 9, 64), (0, 64, 1)),
                                            v_prefix=z(1, 9, 64), k_tail=odd(torch.int16, (1, 1, 5, 64), (7, 0, 64, 1)), v_tail=z(1, 1, 5, 64),
                                            lens=torch.zeros(1, dtype=torch.int32), rows_per_seq=1))
    args = log[-1][1]
    assert (args[4], args[11], args[15], args[16]) == (64, 9 * 64, 5 * 64, 5 * 64)
    b.verify_drafts_dev(**verify_args(target=odd(torch.int32, (1, 2, 50), (0, 60, 1)), tokens=torch.zeros((1, 1), dtype=torch.int64),
                                      randoms=torch.zeros((1, 2), dtype=torch.int64), draft=odd(torch.int32, (1, 1, 50), (0, 0, 1))))
    args = log[-1][1]
    assert (args[2], args[4]) == (60, 50)
