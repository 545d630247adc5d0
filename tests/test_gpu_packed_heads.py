"""examples/decoder_lm.py --packed with any number of heads, and a model that changes
its device between calls."""

import importlib.util
import pathlib

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402

_path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "decoder_lm.py"
_spec = importlib.util.spec_from_file_location("decoder_lm", _path)
decoder_lm = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(decoder_lm)


@pytest.mark.parametrize("heads,d", [(1, 16), (3, 48), (5, 80), (6, 96), (7, 56)])
def test_heads(heads, d):
    model, losses = decoder_lm.train(steps=2, heads=heads, d=d, layers=1, size=4, log=None,
                                     packed=True)
    assert all(loss == loss and abs(loss) < 100 for loss in losses)
    assert heads % model.blocks[0].kv_heads == 0


def test_frequencies_follow_the_ids():
    model = decoder_lm.PackedDecoderLM(32, 64, 4, 2, 1).cuda()
    ids = torch.arange(1, 31, device="cuda")
    offsets = torch.tensor([0, 13, 30], device="cuda")
    want = model(ids, ids, offsets)
    model.frequencies = lm.rotary_frequencies(2 * model.pairs, device="cpu")
    assert torch.equal(model(ids, ids, offsets), want)
    assert model.frequencies.device == ids.device
