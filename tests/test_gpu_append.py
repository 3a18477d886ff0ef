"""vi_norm_rotate_append against its definition in 64 bits.

Tolerance: one rounding to the element type (half a unit in the last place) and
fp32 arithmetic before it: the mean of d squares (d + 2 roundings), the root and
quotient, the weight, and a rotation's two products and sum, in all at most
(d / 2 + 12) x 2^-24 of the pair's magnitude."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FLAG_ERROR = -(1 << 31)
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def turned(x, weight, eps, cos, sin, interleaved):
    """(values, magnitudes of their pairs) in float64; x [rows, heads, d], cos / sin [rows, half]."""
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * weight
    half = cos.shape[1]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out, big = x.copy(), np.abs(x)
    c, s = cos[:, None], sin[:, None]
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    big[..., a] = big[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return out, big


def close(got, want, big, dtype, d, what):
    bound = UNIT[dtype] * np.abs(want) + (d / 2 + 12) * 2.0 ** -23 * big + TINY[dtype]
    assert (np.abs(got - want) <= bound).all(), what


CASES = [   # counts, contexts, heads, kv_heads, dim, rotary, interleaved, page, layout, norm, positions
    ([1], [0], 1, 1, 16, 16, False, 16, "heads", True, False),
    ([1, 1, 1], [15, 16, 31], 4, 2, 64, 64, False, 16, "heads", True, False),
    ([3, 0, 17, 1], [5, 9, 30, 63], 6, 2, 128, 128, False, 32, "heads", True, True),
    ([2, 5], [0, 100], 8, 8, 128, 32, True, 16, "tokens", True, True),
    ([17, 4], [1000, 3], 24, 4, 256, 64, True, 64, "heads", True, False),
    ([7], [2], 3, 1, 80, 48, False, 16, "tokens", True, False),     # threads of a head that hold no chunks
    ([40], [0], 4, 4, 512, 512, False, 256, "heads", True, False),
    ([5, 6], [7, 8], 5, 5, 96, 0, False, 16, "heads", False, False),   # keys and values written as they are
    ([300], [0], 9, 3, 128, 128, True, 16, "heads", True, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_against_the_definition(dev, rng, dtype, case):
    import voidinfer_amd as vi
    counts, context, heads, hk, d, rotary, interleaved, ps, layout, norm, free = case
    lanes, rows = len(counts), sum(counts)
    print("append", dtype, case, flush=True)
    width = max(-(-(c + n) // ps) for c, n in zip(context, counts)) + 1
    pages = lanes * width + 2
    tables = rng.permutation(pages)[:lanes * width].reshape(lanes, width).astype(np.int32)

    def rand(*shape, scale=1.0, offset=0.0):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * scale + offset).to(dtype)

    pad = 8 if rows % 2 else 0     # rows of a wider projection
    qkv = rand(rows, (heads + 2 * hk) * d + pad, scale=2.0).to(dev)
    q, k, v = (x.view(rows, n, d) for x, n in zip(qkv[:, :(heads + 2 * hk) * d].split([heads * d, hk * d, hk * d], 1), (heads, hk, hk)))
    pool = rand(2, pages, hk, ps, d).to(dev) if layout == "heads" else rand(2, pages, ps, hk, d).to(dev).transpose(2, 3)
    angles = rng.uniform(0, 6.28, (max(context) + max(counts) + 3, rotary // 2))
    cos, sin = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    wq, wk = rand(d, offset=1.0, scale=0.3), rand(d, offset=1.0, scale=0.3)
    at = np.concatenate([np.arange(c, c + n) for c, n in zip(context, counts)]).astype(np.int64)
    lane = np.repeat(np.arange(lanes), counts)
    pos = rng.integers(0, len(angles), rows).astype(np.int32) if free else at
    i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=dev)  # noqa: E731
    kw = dict(q_weight=wq.to(dev), k_weight=wk.to(dev)) if norm else {}
    if free:
        kw["positions"] = i32(pos)
    if rotary:
        kw |= dict(cosines=torch.from_numpy(cos).to(dev), sines=torch.from_numpy(sin).to(dev))
    flags = i32([9] * rows)
    before = pool.cpu().double().numpy()
    offs = np.concatenate([[0], np.cumsum(counts)])
    out = vi.norm_rotate_append(q, k, v, pool[0], pool[1], i32(tables), i32(offs), i32(context), eps=1e-5,
                                interleaved=interleaved, flags=flags, **kw)
    assert not flags.any()
    f64 = lambda x: x.double().cpu().numpy()  # noqa: E731
    c64, s64 = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
    want, big = turned(f64(q), f64(wq) if norm else None, 1e-5, c64, s64, interleaved)
    close(f64(out), want, big, dtype, d, "queries")
    want, big = turned(f64(k), f64(wk) if norm else None, 1e-5, c64, s64, interleaved)
    got = f64(pool)
    page, place = tables[lane, at // ps], at % ps
    close(got[0][page, :, place], want, big, dtype, d, "keys")
    assert np.array_equal(got[1][page, :, place], f64(v))
    got[:, page, :, place] = before[:, page, :, place]
    assert np.array_equal(got, before), "nothing else is written"
    # in place, and the same bits again
    again = vi.norm_rotate_append(q, k, v, pool[0], pool[1], i32(tables), i32(offs), i32(context), eps=1e-5,
                                  interleaved=interleaved, out=q, **kw)
    assert again is q and torch.equal(q, out)


def test_rows_that_cannot_be_placed(dev, rng):
    """No page, a page id out of range, an index past the table, an angle out of range: NaN queries, no page
    touched, VI_FLAG_ERROR; the other rows and the padding rows are as they should be."""
    import voidinfer_amd as vi
    i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=dev)  # noqa: E731
    rows = 9
    x = torch.from_numpy(rng.standard_normal((3, rows, 2, 32)).astype(np.float32)).to(dev).to(torch.bfloat16)
    pool = torch.zeros(2, 4, 2, 16, 32, dtype=torch.bfloat16, device=dev)
    out = torch.full_like(x[0], 7)
    flags = i32([5] * rows)
    cos = torch.ones(40, 16, device=dev)
    tables = i32([[0, -1], [4, 1], [2, 3], [-7, 0]])
    # lane 0: rows at 15 (placed) and 16 (no page); lane 1: page 4 of 4; lane 2: 31 and past its table; lane 3: page -7
    vi.norm_rotate_append(x[0], x[1], x[2], pool[0], pool[1], tables, i32([0, 2, 3, 5, 7]), i32([15, 0, 31, -1]), cos,
                          cos * 0, positions=i32([0, 1, 2, 39, 4, 40, -1, 0, 0]), out=out, flags=flags)
    bad = [False, True, True, False, True, True, True]
    assert flags.tolist() == [FLAG_ERROR if b else 0 for b in bad] + [5, 5]
    for r, b in enumerate(bad):
        assert bool(torch.isnan(out[r]).all()) == b and (b or torch.equal(out[r], x[0, r]))
    assert bool((out[7:] == 7).all())
    want = torch.zeros_like(pool)
    want[0, 0, :, 15], want[1, 0, :, 15] = x[1, 0], x[2, 0]
    want[0, 3, :, 15], want[1, 3, :, 15] = x[1, 3], x[2, 3]
    assert torch.equal(pool, want)


def test_zero_and_nonfinite_heads(dev):
    """A head of zeros stays zero (eps keeps the quotient finite); NaN and Inf stay within their head."""
    import voidinfer_amd as vi
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    x = torch.ones(3, 4, 64, dtype=torch.float16, device=dev)
    x[0, 0], x[0, 1, 5], x[1, 2, 63], x[2, 3] = 0, float("nan"), float("inf"), 60000.0
    pool = torch.zeros(2, 1, 4, 16, 64, dtype=torch.float16, device=dev)
    w = torch.ones(64, dtype=torch.float16, device=dev)
    out = vi.norm_rotate_append(x, x, x, pool[0], pool[1], i32([[0]]), i32([0, 3]), i32([0]), q_weight=w, k_weight=w)
    o = out.float()
    assert not o[0, 0].any() and bool(torch.isnan(o[0, 1]).all()) and bool(torch.isnan(o[1, 2, 63]))
    o[0, 0], o[0, 1], o[1, 2] = 1, 1, 1
    assert bool((o == 1).all())              # x / sqrt(mean x^2): squares past fp16's range are fp32's
    assert torch.equal(pool[0, 0].transpose(0, 1)[:3].isnan(), out.isnan())


def test_refusals(dev):
    import voidinfer_amd as vi
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    x = torch.zeros(2, 4, 64, dtype=torch.float16, device=dev)
    pool = torch.zeros(2, 3, 2, 16, 64, dtype=torch.float16, device=dev)
    k = x[:, :2]
    base = (x, k, k, pool[0], pool[1], i32([[0, 1]]), i32([0, 2]), i32([0]))
    vi.norm_rotate_append(*base)
    cos = torch.zeros(8, 32, device=dev)
    for at, bad in ((0, x.float()), (0, x[..., :32]), (1, x), (2, x.bfloat16()), (3, pool[0].transpose(2, 3)), (4, pool[0, :2]),
                    (5, i32([0, 1])), (6, i32([0, 1, 2])), (7, i32([0, 0])), (7, torch.zeros(1, device=dev))):
        args = list(base)
        args[at] = bad
        with pytest.raises(ValueError):
            vi.norm_rotate_append(*args)
    for kw in (dict(cosines=cos), dict(sines=cos), dict(cosines=cos, sines=cos.double()), dict(cosines=cos, sines=cos[:4]),
               dict(q_weight=torch.zeros(64, device=dev)), dict(k_weight=x[0, 0, :32]), dict(out=x[:1]), dict(flags=i32([0])),
               dict(cosines=cos, sines=cos, positions=i32([0])), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            vi.norm_rotate_append(*base, **kw)
