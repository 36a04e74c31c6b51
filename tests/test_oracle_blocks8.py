"""The 8-bit block oracle against facts that do not come from it: torch's own e4m3 rounding, the borders of a block's scale, and
the gradients against differences."""
import torch

from oracle import blocks8 as o


def test_scale_is_the_smallest_power_that_fits():
    for top, s in ((448.0, 0), (448.0000001, 1), (449.0, 1), (224.0, -1), (1.0, -8), (0.0, 0), (896.0, 1), (1e-45, -126), (3.0e38, 120)):
        assert o.exponents(torch.tensor([[top, -top / 2]], dtype=torch.float64)).item() == s


def test_values_are_torchs_e4m3_of_the_scaled_value():
    g = torch.Generator().manual_seed(0)
    v = (torch.randn((7, 300), generator=g) * torch.exp(torch.randn(300, generator=g))).bfloat16().float()
    v[0, :128] = torch.arange(128) * 0.5          # ties
    v[1, 130] = 0
    s = o.exponents(v).repeat_interleave(128, 1)[:, :300]
    ref = torch.ldexp(torch.ldexp(v, -s.int()).to(torch.float8_e4m3fn).float(), s.int())
    assert torch.equal(o.values(v), ref.double())
    bad = v.clone()
    bad[2, 5], bad[3, 200], bad[4, 0] = float("inf"), float("nan"), float("-inf")
    h = o.values(bad)
    assert torch.equal(torch.isnan(h), ~bad.isfinite())
    assert torch.equal(h[0], o.values(v)[0])


def test_square_blocks_of_a_transposed_weight_are_the_transposed_ones():
    w = torch.randn((200, 300), generator=torch.Generator().manual_seed(1))
    assert torch.equal(o.values(w, True).t(), o.values(w.t().contiguous(), True))


def test_half_a_step_bounds_the_error():
    v = torch.randn((50, 128), generator=torch.Generator().manual_seed(2)).double()
    unit = torch.pow(2.0, o.exponents(v))
    assert bool(((o.values(v) - v).abs() <= torch.maximum(v.abs() * 2.0 ** -4, unit * 2.0 ** -10)).all())


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (torch.randn((3, 24), generator=g, dtype=torch.float64) for _ in range(4))
    w, b, h = w[0], b[0], 1e-6
    xh, r = o.ln_parts(x, 1e-6)
    dx, dyxh = o.ln_grads(dy, xh, r, w)

    def f(x, w, b):
        return ((o.ln_parts(x, 1e-6)[0] * w + b) * dy).sum().item()
    for i, j in ((0, 0), (1, 7), (2, 23)):
        d = torch.zeros_like(x)
        d[i, j] = h
        assert abs((f(x + d, w, b) - f(x - d, w, b)) / (2 * h) - dx[i, j].item()) < 1e-7
        assert abs((f(x, w + d[i], b) - f(x, w - d[i], b)) / (2 * h) - dyxh.sum(0)[j].item()) < 1e-7
    t = torch.linspace(-8, 8, 101, dtype=torch.float64)
    assert ((o.gelu(t + h) - o.gelu(t - h)) / (2 * h) - o.gelu_slope(t)).abs().max() < 1e-8
    assert (o.gelu(t) - torch.nn.functional.gelu(t, approximate="tanh")).abs().max() < 1e-12


def test_values_at_the_top_of_the_range_stay_finite():
    """248 * 2^120 lies half way between 240 and 256 steps of 2^120, of which the latter is 2^128."""
    v = torch.tensor([[3.39e38, -3.39e38, 248 * 2.0 ** 120, 247.9 * 2.0 ** 120, 3.0e38]], dtype=torch.float64)
    assert (o.values(v) / 2.0 ** 120).tolist() == [[240.0, -240.0, 240.0, 240.0, 224.0]]
