"""Beam selection with all that it reads and writes side by side in one buffer."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer
from test_gpu_beam import clear_case, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,beams,vocab", [(3, 4, 1000), (1, 8, 60001)])
def test_in_one_buffer(dev, batch, beams, vocab, in_place):
    fin = i32(np.arange(batch * beams).reshape(batch, beams) % 5 == 4)
    c = clear_case(vocab, batch, beams, vocab, beams, finished=fin, end=7)
    size = 4 * batch * beams
    whole = DeviceBuffer(8 * size)
    whole.upload(np.full(whole.nbytes, 0xff, np.uint8))
    scores, finished, *outs, behind = [whole.view(i * size, size, t, (batch, beams)) for i, t in enumerate(
        [np.float32, np.int32, np.int32, np.int32, np.float32, np.int32, np.uint32])]
    scores.upload(c.scores)
    finished.upload(fin)
    if in_place:
        outs[2:] = [scores, finished]
    c.bufs["scores"], c.kw["finished"], c.out = scores, finished, outs
    c.run()
    c.check()
    assert np.all(behind.download() == 0xffffffff)
    if not in_place:
        assert np.array_equal(scores.download(), c.scores) and np.array_equal(finished.download(), fin)
