"""GPU tests of the workspaces that attention over split keys takes: many graphs of one bound stream, two captures of one stream at
a time, and what is refused."""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from test_gpu_paged import Setup

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


def _batches(s, n):
    """Queries and results of n calls, and where they are on the device."""
    w = s.heads * s.dim
    qs = [s.random_bits(s.rows, w) for _ in range(n)]
    want = [s.attend(q=q) for q in qs]
    return qs, want, [s.hip.put(q) for q in qs], [s.hip.alloc(want[0].nbytes) for _ in qs]


def test_many_graphs_share_the_workspace_of_a_bound_stream(hip):
    """Twelve graphs and eager calls in order on one stream, with one workspace."""
    s = Setup(hip, [(9000, 1), (2000, 1)], one_row=True, streams=1)
    s.upload()
    qs, want, dq, do = _batches(s, 12)
    s.op.release()   # (the default stream's)
    st = hip.stream()
    s.op.bind(st, 0)
    call = lambda i: s.op.attend(s.batch, s.kc, s.vc, dq[i], do[i], stream=st)   # noqa: E731
    graphs = [hip.capture(st, lambda i=i: call(i)) for i in range(12)]
    for turn in range(4):
        for p, y in zip(do, want):
            hip.write(p, np.zeros_like(y))
        hip.sync()
        for i in range(12):
            if (i + turn) % 3:
                hip.launch(graphs[i], st)
            else:
                call(i)
        for i in range(12):
            assert np.array_equal(hip.get(do[i], want[i]), want[i]), (turn, i)


def test_two_captures_of_one_stream_at_once(hip):
    """Each capture has a workspace of its own: the graphs run on other streams at the same time."""
    s = Setup(hip, [(9000, 1), (7000, 1)], one_row=True, streams=3)
    s.upload()
    qs, want, dq, do = _batches(s, 2)
    st = [hip.stream() for _ in range(3)]
    graphs = [hip.capture(st[0], lambda i=i: s.op.attend(s.batch, s.kc, s.vc, dq[i], do[i], stream=st[0])) for i in range(2)]
    for turn in range(20):
        for i in range(2):
            hip.launch(graphs[i], st[1 + i])
        if turn % 5 == 4:
            for i in range(2):
                assert np.array_equal(hip.get(do[i], want[i]), want[i]), (turn, i)
                hip.write(do[i], np.zeros_like(want[i]))
    from instantllm_amd.engine import IllError
    with pytest.raises(IllError, match="ill_paged_bind"):   # (the default stream's and the captures' are all there are)
        s.op.attend(s.batch, s.kc, s.vc, dq[0], do[0], stream=st[1])


def test_bindings_refused_and_undone(hip):
    from instantllm_amd.engine import ILL_E_ARG, IllError
    s = Setup(hip, [(9000, 1)], one_row=True, streams=2)
    s.upload()
    qs, want, dq, do = _batches(s, 1)   # (on the default stream: workspace 0)
    st = [hip.stream() for _ in range(3)]

    def call(stream):
        hip.write(do[0], np.zeros_like(want[0]))
        s.op.attend(s.batch, s.kc, s.vc, dq[0], do[0], stream=stream)
        assert np.array_equal(hip.get(do[0], want[0]), want[0])
    for bad, what in (((st[0], 0), "held"), ((None, 0), "held"), ((st[0], 2), "workspace 2 of 2"), ((st[0], -2), "workspace -2"), ((2, 1), "per-thread")):
        with pytest.raises(IllError, match=what) as e:
            s.op.bind(*bad)
        assert e.value.code == ILL_E_ARG
    s.op.bind(st[0], 1)
    s.op.bind(st[1], 1)
    with pytest.raises(IllError, match="bound to workspace 1"):
        s.op.bind(st[1], 0)
    for stream in (st[0], st[1], None):
        call(stream)
    with pytest.raises(IllError, match="as many"):
        s.op.attend(s.batch, s.kc, s.vc, dq[0], do[0], stream=st[2])
    hip.sync()
    s.op.bind(None, None)
    call(st[2])                     # takes what was the default stream's
    with pytest.raises(IllError, match="as many"):
        s.op.attend(s.batch, s.kc, s.vc, dq[0], do[0])
    s.op.bind(st[0], None)
    s.op.bind(st[1], None)
    call(None)
    s.op.release()
    s.op.bind(st[2], 0)
    call(st[2])
    call(st[0])
