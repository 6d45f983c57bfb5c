"""Models of real classes through the call that users make, ``install_paged_attention(model, cache)`` with the model's own
rotation, against the same model without the cache in fp32."""
import copy

import pytest
import torch

from mindpipe_b200 import install, ops
from mindpipe_b200.attention import PagedKVCache
from tests.test_paged_install_cpu import LLAMA3, build

pytestmark = pytest.mark.gpu
TOL = {torch.float16: 1e-2, torch.bfloat16: 8e-2}      # relative Frobenius error of logits: as the linears' tests allow; roundings eight times as large


@pytest.mark.parametrize("kind,settings", [
    ("llama", dict(head_dim=64, rope_parameters=LLAMA3)), ("mistral", dict(sliding_window=128)), ("granite", dict(attention_multiplier=0.03)),
    ("nemotron", dict(partial_rotary_factor=0.5, head_dim=128)), ("qwen2", dict(num_key_value_heads=1))])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@torch.no_grad()
def test_prompts_then_tokens_of_real_models(kind, settings, dtype):
    model = build(kind, **settings).to("cuda", dtype)
    plain = copy.deepcopy(model).float()                          # of the rounded weights
    attn = model.model.layers[0].self_attn
    dim = attn.head_dim
    cache = PagedKVCache(4, 40, 8, attn.k_proj.out_features // dim, dim, dtype=dtype)
    cache.pool.fill_(float("nan"))
    install.install_paged_attention(model, cache)
    g = torch.Generator(device="cuda").manual_seed(1)
    first, more = [90, 1, 33], 12
    sequences = [torch.randint(3, 128, (n + more,), generator=g, device="cuda") for n in first]
    step = cache.prompts(first)
    with cache.running(step):
        logits = model(torch.cat([s[:n] for s, n in zip(sequences, first)])[None], position_ids=step.positions.long()[None],
                       use_cache=False).logits[0]
    got = [[x] for x in logits.split(first)]
    for t in range(more):
        step = cache.next_token(step.sequences)
        with cache.running(step):
            logits = model(torch.stack([s[n + t] for s, n in zip(sequences, first)])[None], position_ids=step.positions.long()[None],
                           use_cache=False).logits[0]
        for mine, x in zip(got, logits):
            mine.append(x[None])
    for mine, s in zip(got, sequences):
        want = plain(s[None], use_cache=False).logits[0].double()
        assert ((torch.cat(mine).double() - want).norm() / want.norm()).item() <= TOL[dtype]
    ops.check_device_errors()
