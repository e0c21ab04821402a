"""The capture hook on this package's attention refuses what that attention does not
compute, instead of dropping it: tiny models on the CPU, the operator replaced."""
import pytest
import torch
from transformers import LlamaConfig, LlamaModel, MistralConfig, MistralModel

from linearard_b200 import distill

IDS = torch.randint(0, 100, (2, 12))


@pytest.fixture
def calls(monkeypatch):
    """Runs the hook with plain attention in the operator's place; what it was given."""
    seen = []

    def plain(q, k, v, mask, causal, scale):
        seen.append((mask, causal, scale))
        G, T = q.shape[1] // k.shape[1], q.shape[2]
        assert k.shape[2] == T, "q/k B/T/D must match"
        s = q @ k.repeat_interleave(G, 1).transpose(-1, -2) * scale
        keep = torch.ones(T, T, dtype=torch.bool)
        keep = keep.tril() if causal else keep
        if mask is not None:
            keep = keep & (mask != 0)[:, None, None, :]
        return s.masked_fill(~keep, -1e9).softmax(-1) @ v.repeat_interleave(G, 1)
    monkeypatch.setattr(distill, "attn", plain)
    return seen


def model(cls, config, impl, **kw):
    torch.manual_seed(0)
    c = config(vocab_size=100, hidden_size=32, intermediate_size=32, num_hidden_layers=2,
               num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=64, **kw)
    c._attn_implementation = impl
    return cls(c).eval()


def both(cls, config, run, **kw):
    """Last hidden states on SDPA and on the package's attention."""
    name = distill.register_capture_attention(attention="own")
    with torch.no_grad():
        return [run(model(cls, config, impl, **kw)).last_hidden_state for impl in ("sdpa", name)]


PACKED = torch.cat([torch.arange(5), torch.arange(7)])[None].repeat(2, 1)


def test_models_without_a_window_run_as_on_sdpa(calls):
    pad = torch.ones(2, 12, dtype=torch.int64)
    pad[1, 8:] = 0
    for cls, config, kw in ((LlamaModel, LlamaConfig, {}),
                            (MistralModel, MistralConfig, dict(sliding_window=None)),
                            (MistralModel, MistralConfig, dict(sliding_window=12)),
                            (MistralModel, MistralConfig, dict(sliding_window=4096))):
        a, b = both(cls, config, lambda m: m(input_ids=IDS, use_cache=False), **kw)
        torch.testing.assert_close(a, b)
        a, b = both(cls, config, lambda m: m(input_ids=IDS, attention_mask=pad, use_cache=False), **kw)
        torch.testing.assert_close(a[pad.bool()], b[pad.bool()])
    assert all(causal for _, causal, _ in calls)


@pytest.mark.parametrize("window", [1, 4, 11])
@pytest.mark.parametrize("pad", [False, True])
def test_a_window_narrower_than_the_sequence_is_refused(calls, window, pad):
    mask = torch.ones(2, 12, dtype=torch.int64) if pad else None
    if pad:
        mask[1, 8:] = 0
    with pytest.raises(AssertionError, match="window|mask"):
        both(MistralModel, MistralConfig,
             lambda m: m(input_ids=IDS, attention_mask=mask, use_cache=False), sliding_window=window)
    assert not calls


def test_packed_sequences_are_refused(calls):
    for cls, config, kw in ((LlamaModel, LlamaConfig, {}),
                            (MistralModel, MistralConfig, dict(sliding_window=4096))):
        with pytest.raises(AssertionError, match="mask"):
            both(cls, config, lambda m: m(input_ids=IDS, position_ids=PACKED, use_cache=False), **kw)
    assert not calls


def test_other_options_of_the_attention_are_refused(calls):
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    f = ALL_ATTENTION_FUNCTIONS[distill.register_capture_attention(attention="own")]

    class Layer:
        layer_idx, is_causal = 0, True
    q, k = torch.randn(1, 4, 6, 8), torch.randn(1, 2, 6, 8)
    f(Layer, q, k, k, None, scaling=0.3, dropout=0.0, sliding_window=None, softcap=None, s_aux=None,
      position_ids=torch.arange(6)[None], use_cache=False)
    f(Layer, q, k, k, None, scaling=0.3, sliding_window=6)
    n = len(calls)
    t = torch.zeros(4)
    for kw in (dict(sliding_window=5), dict(softcap=30.0), dict(s_aux=t), dict(head_mask=t),
               dict(position_bias=t), dict(cu_seq_lens_q=t), dict(cu_seq_lens_k=t), dict(dropout=0.1)):
        with pytest.raises(AssertionError):
            f(Layer, q, k, k, None, scaling=0.3, **kw)
    assert len(calls) == n
