"""The 8-bit cache under the whole-token runner and under transformers' model: what the first attention layer
stores is the quantised form of what the bf16 path stores, code for code (the layers before it see no cache)."""
import pytest
import torch

import kv8_oracle as ora
from conftest import load_pkg
from oracle import lfm2_attention as orc

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
LAYERS = ("conv", "attention", "conv", "attention")


def _state(seed=3, ffn=512, vocab=256):
    kinds = tuple("full_attention" if k == "attention" else k for k in LAYERS)
    return orc.lfm2_model_weights(seed, ffn=ffn, vocab=vocab, layer_types=kinds)


def _runner(dev, **kw):
    mod = load_pkg("lfm2_runner")
    return mod.LFM2DecodeRunner(_state(), mod.LFM2Config(ffn=512, vocab=256, layer_types=LAYERS), max_batch=3,
                                max_context=200, device=dev, **kw)


def _quantised(k, v, chunks):
    """What appending k, v [8, n, 64] in chunks of the given sizes stores, as values."""
    nb = (k.shape[1] + 63) // 64
    f8 = torch.float8_e4m3fn
    c = ora.Cache(torch.zeros(nb, 8, 64, 64).to(f8), torch.zeros(nb, 8, 64, 64).to(f8), torch.ones(nb, 8),
                  torch.ones(nb, 8))
    at = 0
    for n in chunks:
        ora.append(c, list(range(nb)), at, k[:, at:at + n].transpose(0, 1), v[:, at:at + n].transpose(0, 1))
        at += n
    return ora.values(c, list(range(nb)), at)


def test_runner_stores_the_quantised_cache(cuda):
    """Graph, eager and blocks on demand agree bit for bit; the first attention layer's cache is the bf16
    runner's, quantised token by token."""
    ids = torch.randint(0, 256, (3, 70), generator=torch.Generator().manual_seed(1))
    full = _runner(cuda)
    full.prefill(ids)
    runs = [_runner(cuda, kv8=True), _runner(cuda, kv8=True, use_graph=False), _runner(cuda, kv8=True, pool_blocks=8),
            _runner(cuda, kv8=True, fused_glue=False, pool_blocks=6)]
    logits = []
    for r in runs:
        for _ in range(2):                      # again after a reset: blocks and scales start afresh
            r.reset()
            r.prefill(ids)
        r.check()
        logits.append(r.logits.clone())
        for seq in range(3):
            k, v = full.kv(0, seq, 69)
            want_k, want_v = _quantised(k.cpu(), v.cpu(), [1] * 70)
            got_k, got_v = r.kv(0, seq, 69)
            if r.fused_glue:
                assert torch.equal(got_k.cpu().double(), want_k) and torch.equal(got_v.cpu().double(), want_v)
    assert torch.equal(logits[0], logits[1]) and torch.equal(logits[0], logits[2])
    assert bool(torch.isfinite(logits[3]).all())


def test_runner_reports_an_exhausted_pool(cuda):
    r = _runner(cuda, kv8=True, pool_blocks=4)
    r.prefill(torch.zeros(3, 64, dtype=torch.long))
    r.check()
    r.step(torch.zeros(3, dtype=torch.long))             # token 65 of three sequences: one block is left
    with pytest.raises(RuntimeError, match="2 tokens got no block"):
        r.check()
    assert r.past.tolist() == [65, 64, 64]                # what was not cached is not attended
    with pytest.raises(ValueError, match="kv8"):
        _runner(cuda, pool_blocks=4)


def test_hf_model_on_the_8_bit_cache(cuda):
    """A prompt, drafted tokens and single tokens through Lfm2ForCausalLM."""
    from transformers import Lfm2Config, Lfm2ForCausalLM
    hf = load_pkg("hf_paged")
    hf.register()
    cfg = Lfm2Config(hidden_size=1024, intermediate_size=512, num_hidden_layers=4, num_attention_heads=16,
                     num_key_value_heads=8, vocab_size=256, norm_eps=1e-5, block_auto_adjust_ff_dim=False,
                     layer_types=["full_attention", "conv", "full_attention", "conv"],
                     rope_parameters={"rope_type": "default", "rope_theta": 1.0e6}, tie_word_embeddings=True)
    cfg._attn_implementation = hf.NAME
    torch.manual_seed(0)
    model = Lfm2ForCausalLM(cfg).to(BF16).eval().to(cuda)
    ids = torch.randint(0, 256, (2, 110), generator=torch.Generator().manual_seed(2)).to(cuda)
    caches = [hf.B200PagedCache(cfg, max_batch_size=2, max_cache_len=128, device=cuda, shuffle_seed=4, kv8=kv8)
              for kv8 in (False, True)]
    chunks, out = [100, 4, 3, 1, 2], []
    with torch.no_grad():
        for c in caches:
            at, got = 0, []
            for n in chunks:
                got.append(model(ids[:, at:at + n], past_key_values=c, use_cache=True).logits)
                at += n
            c.check()
            out.append(torch.cat(got, 1).float())
    assert out[1].shape == out[0].shape and bool(torch.isfinite(out[1]).all())
    for seq in range(2):
        k, v = caches[0].pool.read_dense(0, seq, 110)
        want_k, want_v = _quantised(k.cpu(), v.cpu(), chunks)
        got_k, got_v = caches[1].pool.read_dense(0, seq, 110)
        assert torch.equal(got_k.cpu().double(), want_k) and torch.equal(got_v.cpu().double(), want_v)
