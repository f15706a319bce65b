"""The contexts that attention on the 8-bit cache hands to the models around it: under transformers' model and in the
whole-token runner, of every attention layer, against the cache that the layer holds at that moment."""
import pytest
import torch

import kv8_oracle as ora
from conftest import load_pkg
from oracle import lfm2_attention as orc
from test_kv8_models_gpu import BF16, _runner, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scaling", [None, 0.2])
def test_hf_model_contexts(cuda, scaling):
    """A prompt, drafted tokens and single tokens; the scale is the module's."""
    from transformers import AttentionInterface, Lfm2Config, Lfm2ForCausalLM
    hf = load_pkg("hf_paged")
    hf.register()
    cfg = Lfm2Config(hidden_size=1024, intermediate_size=512, num_hidden_layers=4, num_attention_heads=16,
                     num_key_value_heads=8, vocab_size=256, norm_eps=1e-5, block_auto_adjust_ff_dim=False,
                     layer_types=["full_attention", "conv", "full_attention", "conv"],
                     rope_parameters={"rope_type": "default", "rope_theta": 1.0e6}, tie_word_embeddings=True)
    cfg._attn_implementation = hf.NAME
    torch.manual_seed(1)
    model = Lfm2ForCausalLM(cfg).to(BF16).eval().to(cuda)
    if scaling is not None:
        for layer in model.model.layers:
            if hasattr(layer, "self_attn"):
                layer.self_attn.scaling = scaling
    cache = hf.B200PagedCache(cfg, max_batch_size=2, max_cache_len=128, device=cuda, shuffle_seed=4, kv8=True)
    tables = cache.tables.cpu()
    seen = []

    def checked(module, query, key, value, mask, **kw):
        att = cache.layers[module.layer_idx].att
        n = query.shape[2]
        past = cache.layers[module.layer_idx].get_seq_length() - n
        before = ora.Cache.of(cache.pool.kv8(att))
        out, _ = hf.paged_attention(module, query, key, value, mask, **kw)
        ref = ora.Cache.of(cache.pool.kv8(att))
        for b in range(2):
            ora.append(before, tables[b], past, key[b].transpose(0, 1).cpu(), value[b].transpose(0, 1).cpu())
            q = query[b].transpose(0, 1).cpu()
            ora.check_context(out[b], *ora.attend(ref, tables[b], past, q, 0.125 if scaling is None else scaling),
                              f"layer {module.layer_idx}, tokens {past} to {past + n}, sequence {b}")
        assert before.same_as(cache.pool.kv8(att))
        seen.append((module.layer_idx, past, n))
        return out, None
    ids = torch.randint(0, 256, (2, 110), generator=torch.Generator().manual_seed(2)).to(cuda)
    AttentionInterface.register(hf.NAME, checked)
    try:
        at = 0
        with torch.no_grad():
            for n in (100, 4, 3, 1, 2):
                model(ids[:, at:at + n], past_key_values=cache, use_cache=True)
                at += n
    finally:
        hf.register()
    cache.check()
    assert seen == [(i, p, n) for p, n in ((0, 100), (100, 4), (104, 3), (107, 1), (108, 2)) for i in (0, 2)]


@pytest.mark.parametrize("kw", [{}, {"fused_glue": False}, {"pool_blocks": 8}, {"fused_glue": False, "pool_blocks": 6}])
def test_runner_contexts(cuda, kw):
    w = _state()
    r = _runner(cuda, kv8=True, use_graph=False, **kw)
    attend, seen = r._attend, []

    def checked(att, qkv):
        out = attend(att, qkv)
        if n % 13 in (0, 12):
            cache, tables = ora.Cache.of(r.cache.kv8(att)), r.tables.cpu()
            p = f"model.layers.{(1, 3)[att]}.self_attn."
            q, k, _ = ora.split(qkv.cpu())
            q, _ = orc.norm_rope_qk(q, k, w[p + "q_layernorm.weight"], w[p + "k_layernorm.weight"],
                                    *orc.rope_cos_sin([n] * 3))
            for b in range(3):
                ora.check_context(out[b:b + 1], *ora.attend(cache, tables[b], n, q[b:b + 1]), f"layer {att}, token {n}")
            seen.append((n, att))
        return out
    r._attend = checked
    ids = torch.randint(0, 256, (3, 66), generator=torch.Generator().manual_seed(3))
    for n in range(66):
        r.step(ids[:, n])
    r.check()
    assert seen == [(n, a) for n in range(66) if n % 13 in (0, 12) for a in range(2)]


def test_runner_forms_agree(cuda):
    """The glue as torch operations on blocks on demand and on reserved ones, captured and not: bit for bit."""
    ids = torch.randint(0, 256, (3, 70), generator=torch.Generator().manual_seed(4))
    logits = []
    for kw in ({}, {"use_graph": False}, {"pool_blocks": 6}, {"pool_blocks": 6, "use_graph": False}):
        r = _runner(cuda, kv8=True, fused_glue=False, **kw)
        r.prefill(ids)
        r.check()
        logits.append(r.logits.clone())
    assert all(torch.equal(logits[0], x) for x in logits[1:])
