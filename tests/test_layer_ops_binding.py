"""The Python binding of the transformer-layer operators without a GPU: on which stream it allocates, what it refuses."""
import contextlib

import pytest

import stx

torch = pytest.importorskip("torch")


class Stream:
    device = torch.device("cpu")
    cuda_stream = 1


class Library:
    """Workspace sizes, and calls that do nothing."""

    def __getattr__(self, name):
        return (lambda *a: 4096) if name.endswith("workspace_size") else (lambda *a: 0)


@pytest.fixture
def allocations(monkeypatch):
    """Every tensor that the binding makes, with the stream that was current (None: the caller's)."""
    current, made = [None], []

    @contextlib.contextmanager
    def on(stream):
        current.append(stream)
        yield
        current.pop()

    def recorded(make):
        def call(*a, **k):
            t = make(*a, **k)
            made.append((tuple(t.shape), current[-1]))
            return t
        return call

    monkeypatch.setattr(torch.cuda, "stream", on)
    for name in ("empty", "empty_like", "zeros"):
        monkeypatch.setattr(torch, name, recorded(getattr(torch, name)))
    monkeypatch.setattr(torch.Tensor, "new_empty", recorded(torch.Tensor.new_empty))
    monkeypatch.setattr(stx, "lib", lambda: Library())
    monkeypatch.setattr(stx, "_typed", lambda t, *a: None)
    monkeypatch.setattr(stx, "_launch", lambda *a: None)
    return made


def calls(stream):
    x, w, dh = torch.ones(6, 8), torch.ones(4, 8), torch.ones(6, 4)
    q, pos, b = torch.ones(2, 3, 4, 8), torch.arange(3, dtype=torch.int32), torch.ones(4)
    stats = torch.ones(1, 2, 2, dtype=torch.float64)
    return [
        lambda: stx.rope_scaled(q, pos, stx.rope_params(8), q, stream=stream),
        lambda: stx.rope_scaled_back(q, pos, stx.rope_params(8), q, stream=stream),
        lambda: stx.group_norm_cl(x, 2, stream=stream),
        lambda: stx.group_norm_cl_back(x, x, stats, 2, stream=stream),
        lambda: stx.gated_ff(x, w, w, stream=stream),
        lambda: stx.gated_ff_back(dh, x, w, w, b_gate=b, b_value=b, stream=stream),
    ]


@pytest.mark.parametrize("call", range(6))
def test_new_tensors_belong_to_the_calls_stream(allocations, call):
    stream = Stream()
    for s in (stream, None):
        run = calls(s)[call]
        allocations.clear()
        run()
        assert allocations and all(on is s for _, on in allocations), allocations


def test_statistics_left_out(allocations):
    x = torch.ones(6, 8)
    y, stats = stx.group_norm_cl(x, 2, stats=False)
    assert y.shape == x.shape and stats is None
    assert (1, 2, 2) not in [shape for shape, _ in allocations]


def test_stream_of_another_device():
    stream = Stream()
    stream.device = torch.device("meta")
    with pytest.raises(ValueError, match="stream"):
        stx._launch(lambda *a: 0, torch.ones(1), stream)
