"""Arguments of the log-probabilities at the ends of their ranges, before any launch (no GPU)."""
import pytest
import torch

from maester_amd import _lib, gemma_layers, linear_token_logprobs
from maester_amd.gemma_layers import GemmaLayerConfig, GemmaTextModel
from maester_amd.token_logprobs import check_softmax_arguments

P = 0x1000


@pytest.mark.parametrize("cap", [1e-50, 1e-45, 1e-39, 9e-31, 2e30, float("inf"), float("nan"), -1e-3])
def test_caps_whose_reciprocal_fp32_cannot_hold(cap):
    with pytest.raises(ValueError, match="softcap"):
        check_softmax_arguments(cap, 1.0)
    if abs(cap) > 1e-46 or cap != cap:                      # (a float argument of 1e-50 is 0, no cap)
        L = _lib.lib()
        assert L.ma_token_logprobs_fwd(P, 10, P, 1, 10, -100, cap, 1.0, 0, P, P, None, None, None, P, 1 << 20, 0, None) == -1
        assert "softcap" in L.ma_last_error().decode()
        assert L.ma_linear_logprobs_fwd(P, 64, P, 64, P, 1, 10, 64, -100, cap, 1.0, P, P, P, P, 1 << 20, 0, None) == -1
        assert "softcap" in L.ma_last_error().decode()


def test_caps_in_range():
    assert [check_softmax_arguments(c, 1.0)[0] for c in (None, 0, 0.0, 1e-30, 30, 1e30)] == [0.0, 0.0, 0.0, 1e-30, 30.0, 1e30]


@pytest.mark.parametrize("chunk", [-1, -300])
def test_negative_blocks(chunk):
    with pytest.raises(ValueError, match="chunk_rows"):
        linear_token_logprobs(torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(4, dtype=torch.long), chunk_rows=chunk)


def test_the_model_hands_its_arguments_on(monkeypatch):
    config = GemmaLayerConfig(dim=256, n_heads=4, num_key_value_heads=2, head_dim=128, max_seq_len=64, sliding_window_size=64,
                              intermediate_size=64, n_layers=1, attn_types=("global",), vocab_size=40)
    with torch.device("meta"):
        model = GemmaTextModel(config)
    seen = []
    monkeypatch.setattr(gemma_layers, "linear_token_logprobs", lambda *a, **kw: seen.append((a, kw)))
    monkeypatch.setattr(model, "_hidden_states", lambda tokens, pos, doc: (tokens, pos, doc))
    model.token_logprobs(1, 2, 3, 4)
    model.token_logprobs(1, 2, 3, 4, temperature=0.5, softcap=30.0, ignore_index=0, chunk_rows=64, filter_ignored=False)
    model.token_logprobs(1, 2, 3, 4, 0.7)
    weight = model.tok_embeddings.weight
    defaults = dict(ignore_index=-100, softcap=None, temperature=1.0, chunk_rows=None, filter_ignored=True)
    assert [(a[0], a[1] is weight, a[2]) for a, _ in seen] == [((1, 3, 4), True, 2)] * 3
    assert [kw for _, kw in seen] == [defaults, dict(ignore_index=0, softcap=30.0, temperature=0.5, chunk_rows=64, filter_ignored=False),
                                      {**defaults, "temperature": 0.7}]
