"""A beam search that ends by an exception leaves nothing of it running on the pool."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from neurogen_b200 import decoding  # noqa: E402
from neurogen_b200.language import LanguageConfig, NativeLanguageModel, SessionPool, init_packed_weights  # noqa: E402


def test_an_exception_waits_for_the_steps_in_flight(monkeypatch):
    """The prompt's steps (hundreds of microseconds each, enqueued in a few) are in flight when the
    selection fails; the pool's next call, on another stream, must not overlap with them."""
    cfg = LanguageConfig()
    model = NativeLanguageModel(cfg, init_packed_weights(cfg, seed=0))
    pool = SessionPool(model, 256)
    pool.step(np.zeros(256, np.int32))   # the step's capture is not part of it
    streams = []
    make = torch.cuda.Stream

    def stream(*args, **kwargs):
        streams.append(make(*args, **kwargs))
        return streams[-1]

    def fails(*args, **kwargs):
        raise RuntimeError('no selection')

    monkeypatch.setattr(torch.cuda, 'Stream', stream)
    monkeypatch.setattr(decoding, 'beam_select', fails)
    with pytest.raises(RuntimeError, match='no selection'):
        pool.beam_search(np.full((64, 100), 7), 4, 3)
    idle = streams[0].query()
    torch.cuda.synchronize()
    assert idle
