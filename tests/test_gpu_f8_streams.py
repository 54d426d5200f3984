"""The layers of test_gpu_f8_layer.py on two streams at once, several passes each.  A
stream does not wait for the host's copies, nor those for it: every pass has buffers of
its own, filled before anything is launched, and every pass is checked."""
import numpy as np
import pytest

from test_gpu_f8_layer import Program

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [(1, 2), (40, 300)])
def test_two_streams_with_passes_of_their_own(px_gpu, rows):
    px = px_gpu
    streams = [px.Stream() for _ in rows]
    passes = [[Program(px, s, M + i) for i in range(5)] for s, M in zip(streams, rows)]
    for p in sum(passes, []):
        p.eu.zero(p.s)  # rows in no group are read by the activation
    for s in streams:
        s.synchronize()
    first = None
    for _ in range(2):
        for p in sum(passes, []):
            p.rng = np.random.default_rng(p.M)
            p.inputs(min(2, p.M))
        for each in zip(*passes):
            for p in each:
                p.launch()
        for s in streams:
            s.synchronize()
        got = [p.check() for p in sum(passes, [])]
        # the same inputs again: the same bits
        if first is not None:
            for a, b in zip(sum(first, ()), sum(got, ())):
                assert np.array_equal(a, b)
        first = [tuple(x.copy() for x in g) for g in got]
    for s in streams:
        s.destroy()
