"""Prompts in portions and conversations in turns: several new tokens behind a polar cache, against the formula in 64 bits."""
import math

import pytest
import torch

from paged_cases import F64, dequantized
from polarquant_amd.modeling_common import PolarConfig
from polarquant_amd.modeling_llama_polar import (LlamaPolarForCausalLM, LlamaPolarGroupAttention, LlamaPolarMixedGroupAttention, LlamaSnapKVAttention)
from polarquant_amd.modeling_qwen_polar import Qwen2PolarGroupAttention
from polarquant_amd.quantize import quantize_and_pack_nbit

pytestmark = pytest.mark.gpu


def _config(n_heads, n_kv, layers=2, **kw):
    return PolarConfig(hidden_size=n_heads * 128, num_attention_heads=n_heads, num_key_value_heads=n_kv, num_hidden_layers=layers, intermediate_size=512,
                       vocab_size=1000, rope_theta=1e4, eos_token_id=[999999], **kw)


def _rope(start, n, dtype, gpu):
    angles = torch.arange(start, start + n, dtype=F64, device=gpu)[:, None] * 1e4 ** (-torch.arange(0, 128, 2, dtype=F64, device=gpu) / 128)
    t = torch.cat([angles, angles], -1)[None]
    return t.cos().to(dtype), t.sin().to(dtype)


def _expected(q, keys, values, sealed, mask, dtype):
    """-> (attention [B, L, N, 128], bound): as tests/paged_cases.py has it, of the last L tokens."""
    B, N, L, _ = q.shape
    Nk, n = keys.shape[1], keys.shape[2]
    u, scale = torch.finfo(dtype).eps / 2, 128 ** -0.5
    k, v = (t.to(F64).repeat_interleave(N // Nk, 1) for t in (keys, values))
    z = torch.matmul(q.to(F64), k.transpose(2, 3).contiguous()) * scale
    seen = torch.arange(n, device=q.device) <= torch.arange(n - L, n, device=q.device)[:, None]
    if mask is not None:
        seen = seen & (mask[:, None, None, :n] != 0)
    p = torch.softmax(z.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
    off = torch.full((n,), 3e-5, dtype=F64, device=q.device)
    off[:sealed] += 2.0 ** -10
    d = scale * q.to(F64).norm(dim=-1) * (k.norm(dim=-1) * off).amax(-1)[..., None]
    y = torch.matmul(p, v)
    tol = torch.matmul(p, v.abs()) * (torch.expm1(2 * d) + u + n * 2.0 ** -23)[..., None] + u * y.abs() + 1e-7
    return y.transpose(1, 2), tol.transpose(1, 2)


@pytest.mark.parametrize("dtype,cls,n_heads,n_kv,options", [
    (torch.float16, LlamaPolarGroupAttention, 4, 2, {}), (torch.bfloat16, LlamaPolarGroupAttention, 4, 4, dict(cache_capacity=128)),
    (torch.bfloat16, Qwen2PolarGroupAttention, 7, 1, dict(rbits=3, tbits=3)), (torch.float16, LlamaPolarGroupAttention, 4, 1, dict(rbits=3, tbits=3, packed_codes=True))])
@pytest.mark.parametrize("turns", [(5, 3, 2), (128, 128, 1, 129), (200, 60, 300, 1, 1, 127), (1, 700)])
@pytest.mark.parametrize("padded", [False, True])
def test_portions_behind_a_cache(gpu, dtype, cls, n_heads, n_kv, options, turns, padded):
    """Each turn sees what is cached as the cache has it, and itself as it is; the cache is what one call for the whole would have made of the same keys."""
    torch.manual_seed(len(turns))
    cfg = _config(n_heads, n_kv, **options)
    att = cls(cfg, 0).to(dtype).to(gpu)
    att.capture, att.o_proj = [], torch.nn.Identity()
    B, total = 2, sum(turns)
    x = (torch.randn(B, total, cfg.hidden_size, device=gpu) * 0.5).to(dtype)
    mask = torch.ones(B, total, dtype=torch.int64, device=gpu)
    mask[1, :min(turns[0] - 1, 150)] = 0
    cache, at, keys, values = None, 0, [], []
    for L in turns:
        before = cache
        if before is not None and before[1] is not None:
            codes = dequantized(tuple(t.clone() for t in before[1:6]), att.rbits, att.tbits, att.packed_codes)
        else:
            codes = torch.empty(B, n_kv, 0, 128, dtype=F64, device=gpu)
        with torch.no_grad():
            out, cache = att(x[:, at:at + L], attention_mask=mask[:, :at + L] if padded else None, past_key_value=cache, position_embeddings=_rope(at, L, dtype, gpu))
        at += L
        q, k, v = att.capture[-1]
        keys.append(k)
        values.append(v)
        assert out.shape == (B, L, n_heads * 128) and cache[-1] == at
        whole = torch.cat(keys, 2)
        sealed = codes.shape[2]
        if before is not None:
            want, tol = _expected(q, torch.cat([codes, whole[:, :, sealed:].to(F64)], 2), torch.cat(values, 2), sealed, mask if padded else None, dtype)
            off = (out.view(B, L, n_heads, 128).to(F64) - want).abs()
            assert bool((off <= tol).all()), float((off / tol).max())
        # the cache: full groups of the keys as they came, the others and the values as they are
        full = at // 128 * 128
        assert torch.equal(cache[6], torch.cat(values, 2))
        assert (cache[0] is None) == (full == at) and (full == at or torch.equal(cache[0], whole[:, :, full:]))
        assert (cache[1] is None) == (full == 0)
        if full:
            for got, one in zip(cache[1:6], quantize_and_pack_nbit(whole[:, :, :full].contiguous(), att.rbits, att.tbits, packed=att.packed_codes)):
                assert torch.equal(got, one)


def test_a_plain_tuple_is_taken_on(gpu):
    """A cache in the reference's format, without the arena that its tensors are views of."""
    cfg = _config(4, 2)
    att = LlamaPolarGroupAttention(cfg, 0).half().to(gpu)
    x = torch.randn(1, 400, cfg.hidden_size, device=gpu).half()
    with torch.no_grad():
        _, cache = att(x[:, :300], past_key_value=None, position_embeddings=_rope(0, 300, torch.float16, gpu))
        plain = tuple(t.clone() if torch.is_tensor(t) else t for t in cache)
        ours, _ = att(x[:, 300:], past_key_value=cache, position_embeddings=_rope(300, 100, torch.float16, gpu))
        theirs, _ = att(x[:, 300:], past_key_value=plain, position_embeddings=_rope(300, 100, torch.float16, gpu))
    assert torch.equal(ours, theirs)


def test_a_conversation(gpu):
    """A model's prompt, its answer token by token, the next turn behind them and an answer to that: every turn reads the layers' caches, and a turn is the same as
    the layers called by hand."""
    torch.manual_seed(3)
    cfg = _config(4, 2, layers=3)
    model = LlamaPolarForCausalLM(cfg).to(torch.bfloat16).to(gpu).eval()
    ids = torch.randint(0, 1000, (2, 333), generator=torch.Generator().manual_seed(1)).to(gpu)
    with torch.no_grad():
        a = model(input_ids=ids[:, :150], num_logits_to_keep=1)
        caches, seen = a.past_key_values, 150
        for _ in range(3):
            caches = model(input_ids=ids[:, seen:seen + 1], past_key_values=caches, num_logits_to_keep=1).past_key_values
            seen += 1
        kept = [tuple(t.clone() if torch.is_tensor(t) else t for t in c) for c in caches]
        b = model(input_ids=ids[:, seen:], past_key_values=caches, num_logits_to_keep=2)
        assert b.logits.shape == (2, 2, 1000) and all(c[-1] == 333 for c in b.past_key_values)
        x = model.model.embed_tokens(ids[:, seen:])
        rope = model.model.rotary_emb(x, torch.arange(seen, 333, device=gpu)[None])
        for layer, cache in zip(model.model.layers, kept):
            x, _ = layer(x, position_embeddings=rope, past_key_value=cache)
        assert torch.equal(model.lm_head(model.model.norm(x)[:, -2:]), b.logits)
        c = model(input_ids=b.logits[:, -1:].argmax(-1), past_key_values=b.past_key_values, num_logits_to_keep=1)
        assert bool(torch.isfinite(c.logits).all()) and c.past_key_values[0][-1] == 334


@pytest.mark.parametrize("cls,options", [(LlamaPolarMixedGroupAttention, dict(vbits=4)), (LlamaSnapKVAttention, dict(snapkv=True))])
def test_other_variants_refuse(gpu, cls, options):
    """4-bit values and evicted prompts: their caches take a prompt in one call."""
    cfg = _config(4, 2, **options)
    att = cls(cfg, 0).half().to(gpu)
    x = torch.randn(1, 200, cfg.hidden_size, device=gpu).half()
    with torch.no_grad():
        _, cache = att(x[:, :150], past_key_value=None, position_embeddings=_rope(0, 150, torch.float16, gpu))
        with pytest.raises(AssertionError):
            att(x[:, 150:], past_key_value=cache, position_embeddings=_rope(150, 50, torch.float16, gpu))
