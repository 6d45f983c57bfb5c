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


@pytest.mark.parametrize("linears", ["w4a16", "w8a8"])
@torch.no_grad()
def test_real_models_with_quantised_linears_are_asked_too(linears):
    """The installers of the linears first: the attention's code is the same, whatever its projections are."""
    model = build("llama", hidden_size=256, head_dim=64, intermediate_size=512).to("cuda", torch.float16)
    if linears == "w4a16":
        install.real_quantize_model_weight(model, 4, {"zero_point": True, "q_group_size": 128})
    else:
        install.quantize_model(model, weight_bits=8, activation_bits=8, act_quant="per_token")
    ids = torch.randint(3, 128, (40,), generator=torch.Generator().manual_seed(3)).cuda()
    want = model(ids[None], use_cache=False).logits[0].double()
    cache = PagedKVCache(4, 10, 8, 2, 64)
    install.install_paged_attention(model, cache)
    step = cache.prompts([40])
    with cache.running(step):
        got = model(ids[None], position_ids=step.positions.long()[None], use_cache=False).logits[0].double()
    # the same linears on inputs that differ by roundings; W8A8 rounds rows to 8 bits, and a step of a code is 2^-7 of the largest
    assert ((got - want).norm() / want.norm()).item() <= {"w4a16": 1e-2, "w8a8": 5e-2}[linears]
    ops.check_device_errors()
