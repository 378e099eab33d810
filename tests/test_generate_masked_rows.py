"""generate() with rows that have no token left to take: nothing here touches a device."""
import torch

from prime_moment_attention_b200 import model


def test_a_row_without_a_token_looks_up_a_valid_one(monkeypatch):
    """The sampler gives -1 for a row of NaN: -1 stands in the result, and no lookup sees it."""
    m = model.PrimeForCausalLM(model.PrimeConfig(vocab_size=11, hidden_size=16, num_layers=1, num_heads=1, head_dim=16,
                                                 use_recurrence=True))
    seen = []

    def forward(ids, **kw):
        seen.append(ids.clone())
        m.embed_tokens(ids)  # an index outside the table raises here
        return {"logits": torch.zeros(ids.shape[0], ids.shape[1], 11), "states": None}

    monkeypatch.setattr(m, "forward", forward)
    monkeypatch.setattr(model.Sampler, "__call__", lambda s, logits, u: (torch.tensor([3, -1]), None))
    out = m.generate(torch.tensor([[1, 2], [4, 5]]), max_new_tokens=3, uniforms=torch.rand(3, 2))
    assert out.tolist() == [[1, 2, 3, 3, 3], [4, 5, -1, -1, -1]]
    assert [s.tolist() for s in seen[1:]] == [[[3], [0]]] * 3
