"""The whole-token runner on blocks on demand when its pool runs out."""
import pytest
import torch

import kv8_oracle as ora
from conftest import load_pkg
from oracle import lfm2_attention as orc
from test_kv8_models_gpu import _runner, _state

pytestmark = pytest.mark.gpu


def _held(r, seq):
    """Everything the runner keeps of a sequence."""
    n = int(r.past[seq])
    return [r.conv_state[:, seq].clone()] + [x.clone() for a in range(2) for x in r.kv(a, seq, n - 1)]


def _check_last_context(r, seq):
    """The last attention layer's context of the last token, against its cache."""
    n = int(r.past[seq])
    q, k, _ = ora.split(r.qkv[seq:seq + 1].cpu())
    w = _state()
    p = "model.layers.3.self_attn."
    q, _ = orc.norm_rope_qk(q, k, w[p + "q_layernorm.weight"], w[p + "k_layernorm.weight"], *orc.rope_cos_sin([n - 1]))
    cache = ora.Cache.of(r.cache.kv8(1))
    ora.check_context(r.attn[1].out[seq:seq + 1], *ora.attend(cache, r.tables[seq].cpu(), n - 1, q), f"sequence {seq}")


@pytest.mark.parametrize("kw", [{}, {"use_graph": False}, {"fused_glue": False}])
def test_a_refused_token_changes_nothing_and_can_be_tried_again(cuda, kw):
    ids = torch.randint(0, 256, (3, 66), generator=torch.Generator().manual_seed(5))
    r = _runner(cuda, kv8=True, pool_blocks=4, **kw)
    whole = _runner(cuda, kv8=True, **kw)                  # every block reserved
    r.prefill(ids[:, :64])
    whole.prefill(ids[:, :64])
    r.check()
    before = [_held(r, s) for s in range(3)]
    nxt = r.step(ids[:, 64]).clone()                       # one block is left: sequence 0's
    assert r.granted.tolist() == [1, 0, 0] and r.past.tolist() == [65, 64, 64]
    for s in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(before[s], _held(r, s)))
    assert nxt[1:].tolist() == ids[1:, 64].tolist()
    with pytest.raises(RuntimeError, match="2 tokens got no block"):
        r.check()
    # sequence 2 is done; 0 goes on, 1 tries again with the id it was given back
    r.block_tables.release(torch.tensor([False, False, True], device=cuda))
    r.conv_state[:, 2] = 0
    nxt[0] = int(ids[0, 65])
    r.step(nxt)
    assert r.granted.tolist() == [1, 1, 0] and r.past.tolist() == [66, 65, 0]      # 2 and 2 of the 4 blocks
    for t in (64, 65):
        whole.step(ids[:, t])
        s = 1 if t == 64 else 0                            # the sequence whose last token this was
        assert torch.equal(r.conv_state[0, s], whole.conv_state[0, s])
        for x, y in zip(r.kv(0, s, t), whole.kv(0, s, t)):
            assert torch.equal(x, y)
    if kw.get("fused_glue", True):
        for s in range(2):
            _check_last_context(r, s)


def test_refusals_are_counted_once_and_forgotten_by_a_reset(cuda):
    r = _runner(cuda, kv8=True, pool_blocks=2)
    r.step(torch.zeros(3, dtype=torch.long))               # the token that is captured
    with pytest.raises(RuntimeError, match="KV pool exhausted: 1 tokens"):
        r.check()
    r.step(torch.zeros(3, dtype=torch.long))
    r.reset()
    r.check()
    assert r.past.tolist() == [0, 0, 0]


def test_generate_raises_when_the_pool_runs_out(cuda):
    prompt = torch.randint(0, 256, (3, 60), generator=torch.Generator().manual_seed(6))
    r = _runner(cuda, kv8=True, pool_blocks=4)
    with pytest.raises(RuntimeError, match="KV pool exhausted"):
        r.generate(prompt, 8)
    r.reset()
    assert r.generate(prompt, 4).shape == (3, 4)
