"""The plain forms of the 8-bit cache and of attention over pages, against the definitions in 64 bits."""
import numpy as np
import pytest
import torch

from pisceslx_b200.ops import cache as C
from pisceslx_b200.ops import reference as ref

F8 = torch.float8_e4m3fn


def _e4m3_numbers():
    vals = []
    for c in range(127):
        e, m = c >> 3, c & 7
        vals.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return np.array(vals)


@pytest.mark.parametrize("power", [-126, -60, -3, 0, 5, 100, 120])
def test_codes_are_the_nearest_numbers_at_the_smallest_exponent(power):
    g = torch.Generator().manual_seed(power + 200)
    x = (torch.randn(40, 64, generator=g).double() * 2.0 ** power).to(torch.bfloat16)
    x[0, 0] = 448.0 * 2.0 ** min(power, 100)
    codes, byte = ref.fp8_rows(x)
    numbers = _e4m3_numbers()
    assert numbers.max() == 448.0
    for r in range(x.shape[0]):
        row = x[r].double().numpy()
        top = np.abs(row).max()
        e = int(byte[r]) - 127
        assert top <= 448.0 * 2.0 ** e and (e == -127 or top > 448.0 * 2.0 ** (e - 1))
        y = row * 2.0 ** -e
        near = np.abs(np.abs(y)[:, None] - numbers[None])
        got = codes[r].float().double().numpy()
        assert np.array_equal(np.abs(np.abs(y) - np.abs(got)), near.min(1)) and np.all((got == 0) | (np.sign(got) == np.sign(y)))
        tie = (near == near.min(1, keepdims=True)).sum(1) > 1
        assert np.all(codes[r].view(torch.uint8).numpy()[tie] % 2 == 0)


def test_rows_that_are_not_finite_read_as_nan_and_zeros_as_zero():
    x = torch.randn(4, 64).to(torch.bfloat16)
    x[1, 5], x[2, 9], x[3] = float("inf"), float("nan"), 0
    codes, byte = ref.fp8_rows(x)
    assert byte[1] == 255 and byte[2] == 255 and byte[3] == 0 and byte[0] != 255
    v = ref._fp8_values(codes, byte)
    assert torch.isnan(v[1:3]).all() and not v[3].any() and torch.isfinite(v[0]).all()


def test_write_then_read_keeps_the_promised_precision():
    g = torch.Generator().manual_seed(1)
    T, hk, d = 50, 3, 64
    k, v = (torch.randn(T, hk * d, generator=g).to(torch.bfloat16) for _ in range(2))
    pages = [torch.zeros(4, 16, hk, d).to(F8) for _ in range(2)] + [torch.zeros(4, hk, 16, dtype=torch.uint8) for _ in range(2)]
    slots = torch.randperm(64, generator=g)[:T].int()
    slots[7] = -1
    C.kv_cache_write_fp8(k, v, *pages, slots)
    for x, y in zip((k, v), C.kv_cache_read_fp8(*pages, slots)):
        assert not y[7].any()
        keep = torch.arange(T) != 7
        x, y = x[keep].double().view(-1, hk, d), y[keep].double().view(-1, hk, d)
        top = x.abs().amax(-1, keepdim=True)
        # half a step: 2^-4 of a number, or 2^-10 of the factor 2^E, where the row's largest is over 224 2^E
        assert bool(((x - y).abs() <= torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 / 224 * top)).all())
    with pytest.raises(IndexError):
        C.kv_cache_read_fp8(*pages, torch.tensor([64], dtype=torch.int32))


@pytest.mark.parametrize("new,total", [([1, 1], [7, 40]), ([3, 0, 9], [30, 5, 9]), ([5, 2], [3, 2])])
@pytest.mark.parametrize("window,first", [(None, 0), (1, 0), (4, 2), (16, 30)])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_over_pages(new, total, window, first, fp8):
    g = torch.Generator().manual_seed(3)
    hq, hk, d, block = 4, 2, 64, 16
    pages = sum(-(-n // block) for n in total) + 1
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(new), 4), -1, dtype=torch.int32)
    k, v = (torch.randn(pages, block, hk, d, generator=g) for _ in range(2))
    ks = vs = None
    plain = (k, v)
    if fp8:
        (k, ks), (v, vs) = ref.fp8_rows(k), ref.fp8_rows(v)
        plain = (ref._fp8_values(k, ks), ref._fp8_values(v, vs))
        ks, vs = ks.transpose(1, 2).contiguous(), vs.transpose(1, 2).contiguous()
    for b, n in enumerate(total):
        for p in range(-(-n // block)):
            table[b, p] = order.pop()
    q = torch.randn(sum(new) + 2, hq, d, generator=g)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    got = C.cache_attention(q, k, v, table, torch.tensor(total, dtype=torch.int32), cu, max(new), window=window, first_tokens=first, k_scale=ks, v_scale=vs)
    assert not got[sum(new):].any()
    row = 0
    for b, (m, n) in enumerate(zip(new, total)):
        for i in range(m):
            pos = n - m + i
            want = torch.zeros(hq, d, dtype=torch.float64)
            seen = [j for j in range(n) if j <= pos and (window is None or j > pos - window or j < first)]
            for h in range(hq):
                if seen:
                    at = [(int(table[b, j // block]), j % block) for j in seen]
                    kk = torch.stack([plain[0][p, o, h // 2] for p, o in at]).double()
                    vv = torch.stack([plain[1][p, o, h // 2] for p, o in at]).double()
                    want[h] = torch.softmax(kk @ q[row, h].double() / d ** 0.5, 0) @ vv
            assert torch.allclose(got[row].double(), want, atol=1e-5, rtol=1e-5)       # sums of 64 products in 32 bits
            row += 1


def test_refusals():
    z = torch.zeros(1, 2, 64)
    page = torch.zeros(1, 16, 1, 64)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        C.cache_attention(z, page, page, torch.zeros(1, 1, dtype=torch.int32), one, window=0)
    with pytest.raises(IndexError):
        C.cache_attention(z, page, page, torch.full((1, 1), 3, dtype=torch.int32), one)
