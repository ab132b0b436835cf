"""A paged engine's arguments without a GPU."""
import pytest
import torch

from syrinx_amd import SxqError
from syrinx_amd import decoder as D

CFG = D.cosyvoice2_lm_config(n_layers=1, max_seq=64)


@pytest.mark.parametrize("cls", [D.DecoderLM, D.SlowAr, D.Qwen2Lm])
@pytest.mark.parametrize("kw", [dict(kv_dtype=torch.bfloat16), dict(kv_dtype=torch.float16), dict(page_size=64, kv_dtype=torch.bfloat16)])
def test_a_cache_that_is_not_paged_holds_f32(cls, kw):
    with pytest.raises(ValueError, match="kv_pages"):
        cls(CFG, **kw)


@pytest.mark.parametrize("kw", [dict(kv_dtype=torch.float16), dict(kv_dtype=torch.int8), dict(page_size=0), dict(page_size=20)])
def test_a_paged_cache_refuses_other_types_and_sizes(kw):
    with pytest.raises(SxqError):
        D.DecoderLM(CFG, kv_pages=4, **kw)
