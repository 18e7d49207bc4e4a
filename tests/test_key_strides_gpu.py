"""Kernel keys of the paged pools with strides no pool can have: refused when the
key is resolved (a launch divides the pool's size by the page stride)."""
import pytest

pytestmark = pytest.mark.gpu

SHAPE = "q_heads=4&kv_heads=2&head_dim=128&page_size=16&max_pages=4"


@pytest.mark.parametrize("stride", [0, -8, -(1 << 40)])
@pytest.mark.parametrize("key", [
    f"paged_attention?max_batch=2&{SHAPE}", f"paged_attention_output?out=4096&{SHAPE}",
    f"prefill_attention?rows=4&{SHAPE}", f"prefill_attention?rows=4&tables=2&{SHAPE}",
    f"window_attention?max_batch=2&window=8&{SHAPE}",
    f"window_prefill_attention?rows=4&window=8&{SHAPE}",
    f"window_prefill_attention?rows=4&window=8&tables=2&{SHAPE}",
    "move_pages?moves=4&heads=2&head_dim=128&page_size=16"])
def test_keys_refuse_page_strides(tmc, key, stride):
    rt = tmc.Runtime()
    assert rt.resolve(key)
    with pytest.raises(RuntimeError, match="page_stride"):
        rt.resolve(f"{key}&page_stride={stride}")
