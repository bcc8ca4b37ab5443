"""What the calls of a serving step hand to the library, without a GPU: the
library is replaced by a recorder, so that the operands' addresses, strides and
sizes can be held against the memory that the tensors own."""
from __future__ import annotations

import contextlib

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


# ---- the streams of memory that a call allocates ------------------------------------------

class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU."""
    device = property(lambda self: torch.device("cuda", 0))
    recorded = []

    def record_stream(self, stream):
        OnGpu.recorded.append((self.data_ptr(), stream.cuda_stream))


class FakeStream:
    log, torchs, captured = None, 7, ()  # captured: handles

    def __init__(self, handle, device=None):
        self.cuda_stream = handle

    def wait_stream(self, other):
        self.log.append(("wait", self.cuda_stream, other.cuda_stream))


@pytest.fixture
def streams(recorded, monkeypatch):
    """The recorded backend on stream 9 with torch on stream 7; allocations and waits are recorded too."""
    b, log = recorded
    from myelith_amd import backend
    entries = backend.lib()
    entries.myl_stream = lambda ctx: 9
    empty = torch.empty

    def allocate(shape, dtype=None, device=None):
        log.append(("empty", shape))
        return empty(shape, dtype=dtype).as_subclass(OnGpu)
    monkeypatch.setattr(torch, "empty", allocate)
    current = []

    @contextlib.contextmanager
    def on(stream):
        current.append(stream)
        yield
        current.pop()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: current[-1] if current else FakeStream(FakeStream.torchs))
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "ExternalStream", FakeStream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: torch.cuda.current_stream().cuda_stream in FakeStream.captured)
    monkeypatch.setattr(FakeStream, "log", log)
    monkeypatch.setattr(OnGpu, "recorded", [])
    return b, log


def on_gpu(args):
    return {k: v.as_subclass(OnGpu) if isinstance(v, torch.Tensor) else v for k, v in args.items()}


def calls_of(b):
    """Each call with its arguments, and its outputs as the caller would give them."""
    i16 = lambda *s: torch.zeros(s, dtype=torch.int16)
    space = dict(workspace=torch.zeros(256, dtype=torch.uint8))
    return [(b.linear_w8a16_adapters_dev, on_gpu(adapter_args()), on_gpu(dict(space, out=i16(3, 5)))),
            (b.attention_prefix_dev, on_gpu(attention_args()), on_gpu(dict(space, out=i16(4, 4, 64)))),
            (b.verify_drafts_dev, on_gpu(verify_args()),
             on_gpu(dict(space, accepted=torch.zeros(2, dtype=torch.int32), out=torch.zeros((2, 4), dtype=torch.int64))))]


@pytest.mark.parametrize("torchs,own", [(7, 3), (7, 9), (0, 3)])
def test_allocated_memory_is_written_after_its_last_use(streams, monkeypatch, torchs, own):
    """torch hands out memory whose last use is queued on its current stream: a context on
    another stream waits for that, after the call's allocations and before its launch.  (The
    context's own stream and the null stream wait for each other by themselves.)"""
    b, log = streams
    monkeypatch.setattr(FakeStream, "torchs", torchs)
    b._own_stream = own
    for call, args, given in calls_of(b):
        for left_out in [given, *([k] for k in given)]:
            log.clear()
            OnGpu.recorded.clear()
            call(**args, **{k: v for k, v in given.items() if k not in left_out})
            kinds = [e[0] if e[0] in ("empty", "wait") else "launch" for e in log if not e[0].endswith("_workspace")]
            assert kinds == ["empty"] * len(left_out) + ["wait", "launch"], (call.__name__, list(left_out), kinds)
            assert ("wait", 9, torchs) in log and [s for _, s in OnGpu.recorded] == [9] * len(left_out)
        log.clear()
        call(**args, **given)
        assert len(log) == 1, log  # nothing allocated, nothing to wait for


@pytest.mark.parametrize("torchs,own", [(9, 3), (0, 9)])
def test_allocating_on_an_ordered_stream_waits_for_nothing(streams, monkeypatch, torchs, own):
    """torch's stream itself, and the context's own stream beside the null stream."""
    b, log = streams
    monkeypatch.setattr(FakeStream, "torchs", torchs)
    b._own_stream = own
    for call, args, given in calls_of(b):
        log.clear()
        call(**args)
        assert not [e for e in log if e[0] == "wait"] and not OnGpu.recorded


@pytest.mark.parametrize("captured", [(7,), (9,), (7, 9)])
def test_allocating_while_one_stream_is_captured_is_refused(streams, monkeypatch, captured):
    """The memory or the launch alone would be the graph's; both in one capture are."""
    b, log = streams
    monkeypatch.setattr(FakeStream, "captured", captured)
    for call, args, given in calls_of(b):
        log.clear()
        if len(captured) == 2:
            call(**args)
        else:
            with pytest.raises(ValueError, match="captured"):
                call(**args)
            assert not [e for e in log if e[0].endswith("_dev")]
        call(**args, **given)


def test_another_devices_memory_is_not_tied_to_the_stream(streams):
    """Operands on another device than the context's are refused; what was allocated there is freed as usual."""
    b, log = streams
    assert b._other_stream(torch.device("cuda", 1)) is None and b._other_stream(torch.device("cuda", 0)) is not None


# ---- arguments that would arrive as something else ------------------------------------------

def test_an_empty_table_is_not_the_greedy_check(recorded):
    """An empty tensor has no address, and no table means greedy."""
    b, log = recorded
    with pytest.raises(ValueError, match="table"):
        b.verify_drafts_dev(**verify_args(exp_lut=torch.zeros(0, dtype=torch.int16)))
    b.verify_drafts_dev(**verify_args(exp_lut=None, randoms=None))
    assert log[-1][1][11:13] == (None, 0)  # table, entries


def test_scalars_outside_their_type_are_refused(recorded):
    """A C byte would keep the low bits of them: 270 fractional bits would be 14."""
    b, log = recorded
    cases = [(b.linear_w8a16_adapters_dev, adapter_args, ("act_frac", "mid_frac", "out_frac"), (-1, 256, 2**40)),
             (b.attention_prefix_dev, attention_args, ("score_shift", "lut_shift", "prob_frac"), (-1, 256, 270)),
             (b.attention_prefix_dev, attention_args, ("score_mult",), (-2**63 - 1, 2**63, 2**64))]
    for call, args, names, values in cases:
        for name in names:
            for v in values:
                with pytest.raises(ValueError, match=name):
                    call(**args(**{name: v}))
    b.linear_w8a16_adapters_dev(**adapter_args(act_frac=0, mid_frac=255, out_frac=255))
    b.attention_prefix_dev(**attention_args(score_mult=-2**63, score_shift=255, lut_shift=0, prob_frac=0))
    assert len([e for e in log if e[0].endswith("_dev")]) == 2
