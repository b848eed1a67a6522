"""token_logprobs' errors on logits as a language model's, at the lengths and row counts of each of its launches.

Bound. A row's sums are of terms in (0, 1], each good to 4 2^-24 of itself (the difference from the lane's maximum, the
exponential, the move to the row's maximum). A lane adds at most n = V / 512 / slices + 1 of them, then a wave, a workgroup and
the slices add 6, 8 and 6 partial sums: the largest such sum is off by at most (n + 24) 2^-24 of itself, and rounding errors of
one sign do not come in rows of hundreds: to nearest, they are independent of the terms, and sqrt(n) of them in a row's worth of
512 lanes leaves under sqrt(n / 512) 2^-24; 6 such deviations are allowed (at n = 300, 4.6 2^-24). With the 4 of the terms, 20 of
the joins, the logarithm's own 2 and half a step of a result under 32 (2^-20 = 16 2^-24): 64 2^-24 = 3.8e-6 for the log
probability. The entropy adds the second sum's error, of the same relative size, times that sum over the first, E <= 12 here, of
which the terms of exp and difference weigh |d| <= 12 times each: 64 2^-24 (1 + E / 8), under 9.6e-6. Means over a call's rows
have no error of the rows' sign but the terms' own: a quarter of the bounds."""
import pytest
import torch

from lowbit import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("m,v,dt", [(1, 151936, torch.float16), (3, 151665, torch.float32), (48, 151936, torch.float32), (64, 151665, torch.bfloat16),
                                    (600, 151665, torch.float16), (600, 151936, torch.float32), (700, 32000, torch.bfloat16), (520, 1000, torch.float32)])
def test_errors_stay_at_32_bits(cuda, m, v, dt):
    g = torch.Generator(device="cuda").manual_seed(v + m)
    x = 2.2 * torch.randn(m, v, generator=g, device="cuda") - 2.0
    likely = torch.randint(0, v, (m, 12), generator=g, device="cuda")
    x.scatter_add_(1, likely, 6.0 + 5.0 * torch.rand(m, 12, generator=g, device="cuda"))
    x = x.to(dt)
    logp, entropy, values, ids = ops.ext().token_logprobs(x, likely[:, 0].contiguous(), 8)
    worst = {}
    for i in range(0, m, 64):
        exact = torch.log_softmax(x[i:i + 64].double(), -1)
        p = exact.exp()
        for name, got, want in (("logp", logp, exact.gather(1, likely[i:i + 64, :1])[:, 0]), ("entropy", entropy, -(p * exact).sum(-1)),
                                ("values", values, exact.gather(1, ids[i:i + 64]))):
            worst.setdefault(name, []).append((got[i:i + 64].double() - want).reshape(-1))
    worst = {k: torch.cat(e) for k, e in worst.items()}
    print({k: (float(e.abs().max()), float(e.mean())) for k, e in worst.items()}, flush=True)
    for name, e in worst.items():
        bound = 64 * U * (2.5 if name == "entropy" else 1.0)
        assert float(e.abs().max()) <= bound, (name, float(e.abs().max()))
        if m >= 48:
            assert abs(float(e.mean())) <= bound / 4, (name, float(e.mean()))
