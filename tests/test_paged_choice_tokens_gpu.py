"""The choice for prompts of about as many tokens as make the kernel take one
token more or fewer per CTA: the same lists as the oracle's, on either side."""
import pytest
import torch

from tests.test_paged_blocks_gpu import choose
from tests.test_paged_gpu import DEV, Step, draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [2, 4, 8, 16])
@pytest.mark.parametrize("more", [-1, 0, 1])
@pytest.mark.parametrize("heads,kv_heads", [(16, 4), (8, 8)])
def test_choice_of_a_prompt_that_just_fills_the_gpu(tokens, more, heads, kv_heads):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    total = -(-tokens * sms // kv_heads) + more
    news = [total - 5, 5] if tokens == 4 else [total]
    st = Step([n + 300 for n in news], news, heads, kv_heads, 64, 64, "bf16", seed=tokens)
    st.fill()
    choose(st, draw((total, heads, 64), 96, "bf16").to(DEV), 32, 5, 1, 2)
