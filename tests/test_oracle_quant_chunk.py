"""The 8-bit row format and the chunk attention of the oracle against torch's own
conversions, the rule's defining inequality and closed forms."""
import numpy as np
import torch

from oracle import chunk, quant


def _bf16(x):
    return torch.tensor(x, dtype=torch.float32).to(torch.bfloat16).double().numpy()


def test_codes_are_torch_float8():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    got = quant.decode(codes.numpy())
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    finite = want[~np.isnan(want)]
    assert np.array_equal(quant.decode(quant.encode(finite)), finite)
    # every point between two codes, the ties among them
    grid = np.unique(np.concatenate([(finite[:, None] * f).ravel() for f in (0.97, 1.0, 1.03125, 1.0625, 1.09)]))
    grid = np.concatenate([grid[np.abs(grid) <= 448], np.arange(-64, 65) * 2.0 ** -11])
    got = quant.decode(quant.encode(grid))
    want = torch.tensor(grid, dtype=torch.float32).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(got, want)


def test_scale_is_the_smallest_power_of_two_that_fits():
    rng = np.random.default_rng(0)
    x = _bf16(rng.standard_normal((200, 128)) * 2.0 ** rng.integers(-60, 60, (200, 1)))
    x[0, :] = 0
    x[1, :] = 0
    x[1, 5] = 448.0
    x[2, :] = 0
    x[2, 5] = _bf16(450.0)
    e = quant.scale_exponent(x)
    a = np.abs(x).max(-1)
    assert e[0] == -117 and e[1] == 0 and e[2] == 1
    assert (a <= 448 * np.ldexp(1.0, e)).all() and (a[1:] > 448 * np.ldexp(1.0, e[1:] - 1)).all()
    codes, s = quant.quantise(x)
    back = quant.dequantise(codes, s)
    # half a step of four significant bits, or half the smallest step
    assert (np.abs(back - x) <= np.maximum(2.0 ** -4 * np.abs(x), np.ldexp(1.0, e - 10)[:, None])).all()
    assert np.array_equal(_bf16(back), back)  # a bf16 value


def test_edges_of_the_format():
    big = _bf16(np.full((1, 128), 3.3895313892515355e38))
    codes, s = quant.quantise(big)
    assert s[0] == 247 and np.isinf(quant.dequantise(codes, s)).all()
    tiny = np.zeros((1, 128))
    tiny[0, 0] = 2.0 ** -133
    codes, s = quant.quantise(tiny)
    assert s[0] == 10 and quant.dequantise(codes, s)[0, 0] in (0.0, 2.0 ** -126)
    odd = _bf16(np.ones((1, 128)))
    odd[0, :3] = [np.nan, np.inf, -np.inf]
    codes, s = quant.quantise(odd)
    back = quant.dequantise(codes, s)[0]
    assert np.isnan(back[:3]).all() and (back[3:] == 1).all()


def test_chunk_against_torch_softmax():
    g = torch.Generator().manual_seed(1)
    L, n, Hq, Hkv, D = 7, 5, 4, 2, 16
    q, k, v = (torch.randn(L, h, D, generator=g, dtype=torch.float64) for h in (Hq, Hkv, Hkv))
    kc, vc = (torch.randn(n, Hkv, D, generator=g, dtype=torch.float64) for _ in range(2))
    for b in (0, 1, 3, 4, 100):
        o, spread, _ = chunk.attend(q, k, v, kc, vc, 0.3, b)
        pos = torch.arange(n + L)
        hidden = torch.zeros(L, n + L, dtype=torch.bool) if b == 0 else pos[None, :] // b > pos[n:, None] // b
        kk, vv = (torch.cat(x).repeat_interleave(Hq // Hkv, 1).transpose(0, 1) for x in ((kc, k), (vc, v)))
        s = (q.transpose(0, 1) @ kk.transpose(1, 2) * 0.3).masked_fill(hidden, float("-inf"))
        want = (torch.softmax(s, -1) @ vv).transpose(0, 1)
        assert torch.allclose(torch.from_numpy(o), want, atol=1e-13)
        assert (spread >= np.abs(o) - 1e-12).all()


def test_chunk_rows_that_see_nothing_finite():
    q = np.ones((1, 1, 4))
    k = np.full((1, 1, 4), -np.inf)
    o, _, _ = chunk.attend(q, k, np.ones((1, 1, 4)), np.zeros((0, 1, 4)), np.zeros((0, 1, 4)), 1.0)
    assert (o == 0).all()
    o, _, _ = chunk.attend(q, k, np.ones((1, 1, 4)), np.ones((2, 1, 4)), np.full((2, 1, 4), 3.0), 1.0, keep=[True, False])
    assert (o == 3).all()
