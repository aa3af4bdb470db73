"""What PagedDecoder.generate refuses, before it touches a GPU."""
import pytest
import torch

from mini_tensorrt_b200 import gpt2, paged

CFG = gpt2.GPT2Config(n_layer=1, d_model=64, n_head=2, d_ff=64, vocab=50, n_pos=32)


def decoder():
    d = object.__new__(paged.PagedDecoder)  # without weights, which live on the GPU
    d.cfg, d.dev, d.page_size, d.cache_dtype = CFG, torch.device("cpu"), 16, torch.float32
    return d


@pytest.mark.parametrize("over", [{"chunk": 0}, {"chunk": -1}, {"beams": 0}, {"beams": -2}, {"beams": 33}, {"eos": 50},
                                  {"eos": -2}, {"max_new": 0}, {"max_new": 32}])
def test_generate_refuses(over):
    """chunk=-1, for one, ran no prompt at all and chose tokens from memory as it was."""
    with pytest.raises(ValueError):
        decoder().generate([[1, 2, 3], [4]], **{"max_new": 2, **over})


@pytest.mark.parametrize("requests,beams", [(1025, 1), (33, 32)])
def test_generate_refuses_more_rows_than_a_call_takes(requests, beams):
    with pytest.raises(ValueError):
        decoder().generate([[1]] * requests, 2, beams=beams)
