"""The float64 recurrence gradient against central differences (CPU)."""
import numpy as np
import torch

from tests.recurrence_oracle import recurrence


def test_gradient_formula_matches_differences():
    g = torch.Generator().manual_seed(3)
    B, L, C = 2, 9, 3
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    p = {"x": r(B, L, C), "f": r(B, L, C) * 2, "bias": r(C), "gate": r(B, L, C), "h0": r(B, C)}
    reset = torch.zeros(B, L, dtype=torch.bool)
    reset[0, 4] = reset[1, 0] = True
    dy, dh = r(B, L, C), r(B, C)

    def loss(q):
        o = recurrence(q["x"], q["f"], q["bias"], q["gate"], q["h0"], reset)
        return (o["y"] * dy.numpy()).sum() + (o["h"] * dh.numpy()).sum()

    grads = recurrence(p["x"], p["f"], p["bias"], p["gate"], p["h0"], reset, dy, dh)
    eps = 1e-5  # truncation eps^2 and rounding 1e-16 / eps: both below 1e-9
    for name, t in p.items():
        d = grads["d" + name].reshape(-1)
        for i in range(t.numel()):
            up, down = t.clone(), t.clone()
            up.view(-1)[i] += eps
            down.view(-1)[i] -= eps
            num = (loss({**p, name: up}) - loss({**p, name: down})) / (2 * eps)
            assert abs(num - d[i]) < 1e-7, (name, i, num, d[i])


def test_a_reset_cuts_the_state():
    g = torch.Generator().manual_seed(4)
    x, f = torch.randn(1, 12, 2, generator=g), torch.randn(1, 12, 2, generator=g)
    reset = torch.zeros(1, 12, dtype=torch.uint8)
    reset[0, 5] = 1
    whole = recurrence(x, f, reset=reset)["y"]
    np.testing.assert_allclose(whole[:, 5:], recurrence(x[:, 5:], f[:, 5:])["y"], rtol=0, atol=0)
