"""Passes in 8-bit rows on streams and threads at the same time, over buffers that hold another
input's results or NaN when they begin: a step that does not run, or reads before the step that
writes for it, shows."""
import threading

import pytest
import torch

from test_gpu_a8_pass import Buffers, hip, model, rows, run  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def spoil(s):
    """What a pass writes, as no pass leaves it; the codes and the workspace keep what the last
    pass left there."""
    for t in (s.h, s.mid, s.back, s.logits, s.lp, s.entropy, s.top):
        t.fill_(float("nan"))
    s.ids.fill_(-9)


def expected(hip, model, s, inputs, T):  # noqa: F811
    want = []
    for x, t in inputs:
        spoil(s)
        s.targets.copy_(t)
        run(hip, model, s, x, T)
        want.append(s.outputs())
    for a, b in zip(*want):
        assert not torch.equal(a, b)   # the inputs are told apart by every output
    torch.cuda.synchronize()
    return want


def passes(hip, model, s, inputs, T, count):  # noqa: F811
    """`count` passes on the current stream, the two inputs in turn; their outputs."""
    out = []
    for i in range(count):
        if i % 3 == 1:
            spoil(s)
        x, t = inputs[i % 2]
        s.targets.copy_(t)
        run(hip, model, s, x, T)
        out.append(s.outputs())
    return out


def same(out, want):
    for i, got in enumerate(out):
        for name, a, b in zip(("h", "logits", "lp", "entropy", "ids", "top"), got, want[i % 2]):
            assert torch.equal(a, b), (i, name)


@pytest.mark.parametrize("T", [1, 12, 40, 90, 300])
def test_one_after_another(hip, model, T):  # noqa: F811
    s, inputs = Buffers(hip, T), [rows(T, 400 + i) for i in range(2)]
    want = expected(hip, model, s, inputs, T)
    same(passes(hip, model, s, inputs, T, 6), want)
    torch.cuda.synchronize()
    s.free()


@pytest.mark.parametrize("T", [1, 12, 40, 90, 300])
def test_two_streams(hip, model, T):  # noqa: F811
    streams = [torch.cuda.Stream() for _ in range(2)]
    kept = [Buffers(hip, T) for _ in range(2)]
    inputs = [[rows(T, 500 + 2 * i + j) for j in range(2)] for i in range(2)]
    want = [expected(hip, model, s, x, T) for s, x in zip(kept, inputs)]
    out = [[], []]
    for i in range(8):   # a pass to each stream in turn
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                s, (x, t) = kept[j], inputs[j][i % 2]
                if i % 3 == 1:
                    spoil(s)
                s.targets.copy_(t)
                run(hip, model, s, x, T)
                out[j].append(s.outputs())
    torch.cuda.synchronize()
    for j in range(2):
        same(out[j], want[j])
        kept[j].free()


def test_threads(hip, model):  # noqa: F811
    """Host threads that launch at once, on their own streams and buffers, other row counts."""
    sizes = (9, 40, 24, 1)
    kept = [Buffers(hip, T) for T in sizes]
    inputs = [[rows(T, 600 + 2 * T + j) for j in range(2)] for T in sizes]
    want = [expected(hip, model, s, x, T) for s, x, T in zip(kept, inputs, sizes)]
    errors = []

    def work(T, s, x, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                out = passes(hip, model, s, x, T, 10)
                torch.cuda.current_stream().synchronize()
                same(out, w)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(sizes, kept, inputs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for s in kept:
        s.free()
