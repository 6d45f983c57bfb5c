"""A llama-shaped model whose linears and attention are this package's: prompts and later tokens through the paged cache,
against the same model in 64 bits that sees whole sequences."""
import pytest
import torch
from torch import nn

from mindpipe_b200 import install, ops
from mindpipe_b200.attention import PagedKVCache, rotary_table
from mindpipe_b200.modules import SmoothQuantLinear, VllmPackedInt4Linear
from tests._tiny_llama import TinyLlama

pytestmark = pytest.mark.gpu
TOL = 1e-2          # relative Frobenius error, as the linears' tests allow
DIM, KV_HEADS, HIDDEN = 64, 2, 256


class _Runs(nn.Module):
    """The tiny tree run as a decoder: attention and MLP with residuals."""

    def __init__(self, tree):
        super().__init__()
        self.model = tree.model
        self.model.layers = tree.model.layers

    def forward(self, x):
        for layer in self.model.layers:
            x = x + layer.self_attn(x / x.norm(dim=-1, keepdim=True) * 16)[0]
            y = x / x.norm(dim=-1, keepdim=True) * 16
            x = x + layer.mlp.down_proj(nn.functional.silu(layer.mlp.gate_proj(y)) * layer.mlp.up_proj(y))
        return x


def _weights(linear):
    return linear.dequantize() if isinstance(linear, (VllmPackedInt4Linear, SmoothQuantLinear)) else linear.weight


def _plain(model, x, inv_freq):
    """One whole sequence [tokens, hidden] in 64 bits with the weights the model holds."""
    def lin(m, y):
        b = m.bias
        return y @ _weights(m).double().T + (0 if b is None else b.double())

    n = x.shape[0]
    angle = torch.arange(n, device=x.device, dtype=torch.float64)[:, None] * inv_freq.double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotate(y):
        z = torch.complex(*y.chunk(2, -1)) * turn
        return torch.cat([z.real, z.imag], -1)

    x = x.double()
    for layer in model.model.layers:
        a, y = layer.self_attn, x / x.norm(dim=-1, keepdim=True) * 16
        q, k, v = (lin(p, y).view(n, -1, DIM) for p in (a.q_proj, a.k_proj, a.v_proj))
        q, k = rotate(q), rotate(k)
        k, v = (t.repeat_interleave(q.shape[1] // KV_HEADS, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * DIM ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -torch.inf)
        x = x + lin(a.o_proj, torch.einsum("hqk,khd->qhd", s.softmax(-1), v).reshape(n, -1))
        y = x / x.norm(dim=-1, keepdim=True) * 16
        x = x + lin(layer.mlp.down_proj, nn.functional.silu(lin(layer.mlp.gate_proj, y)) * lin(layer.mlp.up_proj, y))
    return x


def _rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("linears", ["float", "w4a16"])
@pytest.mark.parametrize("page", [8, 24])
@torch.no_grad()
def test_prompts_then_tokens_agree_with_whole_sequences(linears, page):
    tree = TinyLlama(seed=3).cuda()
    if linears == "w4a16":
        install.real_quantize_model_weight(tree, 4, {"zero_point": True, "q_group_size": 128})
    cache = PagedKVCache(2, 60, page, KV_HEADS, DIM)
    cache.pool.fill_(float("nan"))                                # pages begin as garbage
    inv = 10000.0 ** (-torch.arange(DIM // 2, dtype=torch.float64, device="cuda") / (DIM // 2))
    names = install.install_paged_attention(tree, cache, cos_sin=rotary_table(inv, 512))
    assert names == [f"model.layers.{i}.self_attn" for i in range(2)]
    model = _Runs(tree)
    g = torch.Generator(device="cuda").manual_seed(1)
    lens, more = [50, 1, 23], 20
    sequences = [torch.randn(n + more, HIDDEN, generator=g, device="cuda").half() for n in lens]
    step = cache.prompts(lens)
    with cache.running(step):
        out = model(torch.cat([s[:n] for s, n in zip(sequences, lens)]))
    got = [[o] for o in out.split(lens)]
    for t in range(more):
        step = cache.next_token(step.sequences)
        x = torch.stack([s[n + t] for s, n in zip(sequences, lens)])
        with cache.running(step):
            out = model(x[:, None] if t % 2 else x)              # with and without a dimension of one token
        for mine, o in zip(got, out.view(len(lens), 1, -1)):
            mine.append(o)
    for mine, s in zip(got, sequences):
        assert _rel(torch.cat(mine), _plain(model, s, inv)) <= TOL
    ops.check_device_errors()


@torch.no_grad()
def test_captured_decode_step_is_refilled_and_replayed():
    tree = TinyLlama(seed=4).cuda()
    install.real_quantize_model_weight(tree, 4, {"zero_point": True, "q_group_size": 128})
    inv = 10000.0 ** (-torch.arange(DIM // 2, dtype=torch.float64, device="cuda") / (DIM // 2))
    eager, replayed = PagedKVCache(2, 30, 16, KV_HEADS, DIM), PagedKVCache(2, 30, 16, KV_HEADS, DIM)
    table, lens = rotary_table(inv, 512), [17, 40]
    install.install_paged_attention(tree, eager, cos_sin=table)
    model = _Runs(tree)
    g = torch.Generator(device="cuda").manual_seed(2)
    prompt = torch.randn(sum(lens), HIDDEN, generator=g, device="cuda").half()
    tokens = torch.randn(6, 2, HIDDEN, generator=g, device="cuda").half()
    ids = {}
    want = []
    for cache in (eager, replayed):
        for layer in tree.model.layers:
            layer.self_attn.cache = cache
        with cache.running(cache.prompts(lens)) as step:
            ids[cache] = step.sequences
            model(prompt)
    for layer in tree.model.layers:
        layer.self_attn.cache = eager
    for x in tokens:
        with eager.running(eager.next_token(ids[eager])):
            want.append(model(x))
    for layer in tree.model.layers:
        layer.self_attn.cache = replayed
    step, x = replayed.reserve(2, 64), torch.zeros(2, HIDDEN, dtype=torch.float16, device="cuda")
    with replayed.running(step):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model(x)                                              # an empty step: stores nothing
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model(x)
    for t, token in enumerate(tokens):
        replayed.next_token(ids[replayed], into=step)
        x.copy_(token)
        graph.replay()
        assert torch.equal(y, want[t])
    ops.check_device_errors()
