"""Kernels of the paged cache in 8 bits and of attention over pages, against plain math in 64 bits."""
import math

import pytest
import torch

from pisceslx_b200.ops import KernelStatusError, check_status
from pisceslx_b200.ops import cache as C
from pisceslx_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn


def _bits(shape, seed, finite=True):
    """bf16 numbers of every magnitude: random bit patterns."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-32768, 32768, shape, generator=g, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    return torch.where(torch.isfinite(x), x, torch.ones_like(x)) if finite else x


def _empty(blocks, block, hk, d):
    codes = lambda: torch.full((blocks, block, hk, d), 0x11, dtype=torch.uint8, device=DEV).view(F8)
    scale = lambda: torch.full((blocks, hk, block), 77, dtype=torch.uint8, device=DEV)
    return codes(), codes(), scale(), scale()


def _same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


# ------------------------------------------------------------------------------------------------
# writing and reading
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,hk,d,block", [(1, 8, 128, 64), (1, 1, 64, 16), (5, 3, 64, 48), (131, 4, 128, 64), (700, 2, 64, 16),
                                               (3001, 8, 128, 64), (149, 16, 64, 32)])
@pytest.mark.parametrize("kind", ["normal", "bits", "wild"])
def test_write_and_read_match_the_definition_bit_for_bit(tokens, hk, d, block, kind):
    g = torch.Generator().manual_seed(tokens)
    if kind == "normal":
        kv = torch.randn(tokens, 2 * hk * d, generator=g).to(torch.bfloat16)
    else:
        kv = _bits((tokens, 2 * hk * d), tokens, finite=kind == "bits")
        # rows of one magnitude each too, so that codes below the largest are met in every one
        kv[::2] = (torch.randn(kv[::2].shape, generator=g) * torch.exp2(torch.randint(-130, 126, (len(kv[::2]), 1), generator=g).double())
                   ).to(torch.bfloat16)
        if kind == "bits":
            kv = torch.where(torch.isfinite(kv), kv, torch.ones_like(kv))
    if tokens > 2:
        kv[2] = 0
    blocks = -(-tokens // block) + 2
    slots = torch.randperm(blocks * block, generator=g)[:tokens].int()
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]
    mine, plain = _empty(blocks, block, hk, d), tuple(t.cpu() for t in _empty(blocks, block, hk, d))
    dev = kv.to(DEV)
    C.kv_cache_write_fp8(dev[:, :hk * d], dev[:, hk * d:], *mine, slots.to(DEV))
    ref.kv_cache_write_fp8(kv[:, :hk * d], kv[:, hk * d:], *plain, slots)
    for a, b in zip(mine, plain):
        assert _same(a, b)
    back = C.kv_cache_read_fp8(*mine, slots.to(DEV))
    want = ref.kv_cache_read_fp8(*plain, slots)
    for a, b in zip(back, want):
        assert a.shape == (tokens, hk * d) and torch.equal(torch.nan_to_num(a.cpu().float(), nan=-7.0), torch.nan_to_num(b.float(), nan=-7.0))
    check_status()


def test_every_code_and_exponent_is_read_as_its_value():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256).view(4, 128, 1, 128).view(F8)
    scale = torch.arange(256, dtype=torch.uint8).repeat_interleave(2).view(4, 1, 128)
    slots = torch.arange(512, dtype=torch.int32)
    k, v = C.kv_cache_read_fp8(*(t.to(DEV) for t in (codes, codes, scale, scale)), slots.to(DEV))
    want, _ = ref.kv_cache_read_fp8(codes, codes, scale, scale, slots)
    assert torch.equal(torch.nan_to_num(k.cpu().float(), nan=-7.0), torch.nan_to_num(want.float(), nan=-7.0))
    assert torch.equal(torch.nan_to_num(v.cpu().float(), nan=-7.0), torch.nan_to_num(want.float(), nan=-7.0))


def test_rows_at_odd_addresses_are_copied_and_slots_outside_are_reported():
    hk, d = 2, 64
    wide = torch.randn(9, 2 * hk * d + 3, device=DEV).to(torch.bfloat16)
    k, v = wide[:, 1:1 + hk * d], wide[:, 1 + hk * d:1 + 2 * hk * d]
    mine, want = _empty(2, 16, hk, d), _empty(2, 16, hk, d)
    slots = torch.arange(9, dtype=torch.int32, device=DEV)
    C.kv_cache_write_fp8(k, v, *mine, slots)
    C.kv_cache_write_fp8(k.contiguous(), v.contiguous(), *want, slots)
    assert all(_same(a, b) for a, b in zip(mine, want))
    slots[4] = 32
    C.kv_cache_write_fp8(k, v, *mine, slots)
    with pytest.raises(KernelStatusError):
        check_status()
    assert all(_same(a, b) for a, b in zip(mine, want))
    rows, _ = C.kv_cache_read_fp8(*mine, slots)
    with pytest.raises(KernelStatusError):
        check_status()
    assert not rows[4].any()


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def _case(new, total, hq, hk, d, block, fp8, seed=0, spread=1.0, window=None, first=0, dirty=True):
    """Pages in no order; what belongs to no token, and pages that nothing sees, hold NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in total]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=g).tolist()
    table = torch.full((len(total), max(need + [1]) + 1), -1, dtype=torch.int32)
    kv = [torch.full((blocks, block, hk, d), float("nan") if dirty else 0.0, dtype=torch.bfloat16) for _ in range(2)]
    dense = []
    for b, n in enumerate(total):
        x = [(torch.randn(n, hk, d, generator=g) * spread).to(torch.bfloat16) for _ in range(2)]
        for p in range(need[b]):
            page = order.pop()
            hidden = window is not None and (p + 1) * block <= n - new[b] - window + 1 and p * block >= first
            table[b, p] = -1 if hidden else page
            for pool, rows in zip(kv, x):
                part = rows[p * block:(p + 1) * block]
                if not hidden:
                    pool[page, :len(part)] = part
        dense.append(x)
    q = torch.randn(sum(new), hq, d, generator=g).to(torch.bfloat16)
    case = dict(q=q.to(DEV), table=table.to(DEV), lens=torch.tensor(total, dtype=torch.int32, device=DEV), ks=None, vs=None)
    if fp8:
        packed = [ref.fp8_rows(pool) for pool in kv]
        case.update(k=packed[0][0].to(DEV), v=packed[1][0].to(DEV), ks=packed[0][1].transpose(1, 2).contiguous().to(DEV),
                    vs=packed[1][1].transpose(1, 2).contiguous().to(DEV))
        dense = [[ref._fp8_values(*ref.fp8_rows(t)) for t in x] for x in dense]
    else:
        case.update(k=kv[0].to(DEV), v=kv[1].to(DEV))
    case["cu"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    return case, dense


def _oracle(q, dense, new, total, window, first, scale):
    """Output in 64 bits, and the sum of |weight x value|, which roundings of the weights are relative to."""
    hq, d = q.shape[1:]
    q = q.double().to(DEV)
    outs, sizes = [], []
    at = 0
    for (k, v), m, n in zip(dense, new, total):
        hk = k.shape[1]
        o, a = torch.zeros(m, hq, d, dtype=torch.float64, device=DEV), torch.zeros(m, hq, d, dtype=torch.float64, device=DEV)
        if n > 0 and m > 0:
            k, v = k.double().to(DEV).repeat_interleave(hq // hk, 1), v.double().to(DEV).repeat_interleave(hq // hk, 1)
            i, j = torch.arange(n - m, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
            ok = j <= i
            if window is not None:
                ok &= (i - j < window) | (j < first)
            sc = (torch.einsum("mhd,nhd->hmn", q[at:at + m], k) * scale).masked_fill(~ok, float("-inf"))
            w = torch.softmax(sc, -1).masked_fill(~ok.any(1)[None, :, None], 0.0)
            o, a = torch.einsum("hmn,nhd->mhd", w, v), torch.einsum("hmn,nhd->mhd", w, v.abs())
        outs.append(o)
        sizes.append(a)
        at += m
    return torch.cat(outs), torch.cat(sizes)


def _close(got, want, size):
    """Weights are rounded to bf16 (2^-8 of each), the result too (2^-8 of it).  The rest is within 2^-10 of each weight: 2^x to
    1e-4 in numerator and denominator, 128 products summed in 32 bits (128 x 2^-24 of a sum of up to some 40)."""
    bad = (got.double() - want).abs() > (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -8 * want.abs()
    assert not bad.any() and torch.isfinite(got).all(), (int(bad.sum()), float((got.double() - want).abs().max()))


def _run(case, new, **kw):
    return C.cache_attention(case["q"], case["k"], case["v"], case["table"], case["lens"], case["cu"], max(new), k_scale=case["ks"],
                             v_scale=case["vs"], **kw)


SHAPES = [
    # new tokens, cached tokens (these among them)
    ([1], [1]), ([1], [128]), ([1], [129]), ([1, 1, 1], [1, 64, 65]), ([1] * 5, [700, 3, 256, 0, 1025]), ([2], [2]), ([7, 1, 3], [7, 500, 130]),
    ([32], [32]), ([33], [4096]), ([65, 0, 64], [65, 40, 300]), ([128], [128]), ([129, 5], [400, 2000]), ([300, 17, 1, 256], [300, 17, 999, 700]),
    ([513], [1500]), ([5, 4], [3, 4]),
]


@pytest.mark.parametrize("new,total", SHAPES)
@pytest.mark.parametrize("hq,hk,d,block", [(32, 8, 128, 64), (16, 4, 64, 64), (4, 4, 64, 16), (6, 2, 128, 48), (8, 1, 128, 128), (5, 1, 64, 32)])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention(new, total, hq, hk, d, block, fp8):
    case, dense = _case(new, total, hq, hk, d, block, fp8, seed=len(new) + total[0])
    got = _run(case, new)
    check_status()
    _close(got, *_oracle(case["q"], dense, new, total, None, 0, d ** -0.5))


@pytest.mark.parametrize("new,total", [([1, 1], [900, 77]), ([3, 2, 5], [1000, 333, 5]), ([200], [1300]), ([70, 301], [2000, 301]), ([600], [600])])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (64, 0), (100, 4), (128, 130), (257, 64), (700, 300), (5000, 4)])
@pytest.mark.parametrize("fp8,hq,hk,d,block", [(False, 8, 2, 128, 64), (True, 8, 2, 128, 64), (False, 4, 1, 64, 16), (True, 6, 2, 64, 48)])
def test_window_and_first_tokens(new, total, window, first, fp8, hq, hk, d, block):
    case, dense = _case(new, total, hq, hk, d, block, fp8, seed=window + first, window=window, first=first)
    got = _run(case, new, window=window, first_tokens=first)
    check_status()
    _close(got, *_oracle(case["q"], dense, new, total, window, first, d ** -0.5))


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 32])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window,first", [(None, 0), (300, 70)])
@pytest.mark.parametrize("new,total", [([1, 1, 1], [1500, 40, 700]), ([90, 2], [1100, 600])])
def test_key_ranges_join(splits, fp8, window, first, new, total):
    case, dense = _case(new, total, 8, 2, 128, 64, fp8, seed=splits, window=window, first=first)
    got = _run(case, new, window=window, first_tokens=first, splits=splits)
    check_status()
    _close(got, *_oracle(case["q"], dense, new, total, window, first, 128 ** -0.5))


@pytest.mark.parametrize("fp8", [False, True])
def test_many_items_per_block_of_threads(fp8):
    new, total = [400, 31, 257, 1], [2100, 900, 257, 4000]
    case, dense = _case(new, total, 64, 8, 128, 64, fp8)
    got = _run(case, new)
    check_status()
    _close(got, *_oracle(case["q"], dense, new, total, None, 0, 128 ** -0.5))


@pytest.mark.parametrize("spread", [0.0, 8.0])
@pytest.mark.parametrize("fp8", [False, True])
def test_flat_and_peaked_weights(spread, fp8):
    new, total = [3, 140], [2000, 700]
    case, dense = _case(new, total, 8, 2, 128, 64, fp8, spread=spread)
    got = _run(case, new, scale=0.05)
    _close(got, *_oracle(case["q"], dense, new, total, None, 0, 0.05))


@pytest.mark.parametrize("d", [64, 128])
def test_every_code_reaches_the_output_as_its_value(d):
    """One visible key: the output is its value, code by code and exponent by exponent (those whose values bf16 holds as normal
    numbers: from byte 20 on, 2^-9 2^(20 - 127) = 2^-116)."""
    bytes_ = torch.arange(20, 248)
    n = len(bytes_) * (256 // d)
    codes = torch.arange(256, dtype=torch.uint8).repeat(len(bytes_))
    codes[(codes & 0x7F) == 0x7F] = 0                        # the writer's codes are numbers
    pages = torch.zeros(n, 16, 1, d, dtype=torch.uint8)
    pages[:, 0, 0] = codes.view(n, d)
    scale = torch.full((n, 1, 16), 127, dtype=torch.uint8)
    scale[:, 0, 0] = bytes_.repeat_interleave(256 // d).to(torch.uint8)
    keys = torch.zeros(n, 16, 1, d, dtype=torch.uint8)
    one = torch.full((n, 1, 16), 127, dtype=torch.uint8)
    q = torch.randn(n, 1, d).to(torch.bfloat16)
    got = C.cache_attention(q.to(DEV), keys.view(F8).to(DEV), pages.view(F8).to(DEV), torch.arange(n, dtype=torch.int32, device=DEV).view(n, 1),
                            torch.ones(n, dtype=torch.int32, device=DEV), k_scale=one.to(DEV), v_scale=scale.to(DEV))
    want = ref._fp8_values(codes.view(F8).view(n, d), scale[:, 0, 0]).to(torch.bfloat16)
    fits = torch.isfinite(want).all(1)
    assert int(fits.sum()) > n - 20
    assert torch.equal(got[:, 0].cpu()[fits], want[fits])


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_behind_the_last_sequence(fp8):
    new, total = [3, 2], [400, 50]
    case, dense = _case(new, total, 8, 2, 64, 64, fp8)
    want, size = _oracle(case["q"], dense, new, total, None, 0, 64 ** -0.5)
    case["q"] = torch.cat([case["q"], torch.full_like(case["q"], float("nan"))])
    got = _run(case, new)
    _close(got[:5], want, size)
    assert not got[5:].any()
    for splits in (1, 4):
        wide = torch.full((10, 2 * 8 * 64), 3.0, dtype=torch.bfloat16, device=DEV)
        out = wide[:, 8 * 64:].view(10, 8, 64)
        assert _run(case, new, out=out, splits=splits).data_ptr() == out.data_ptr()
        _close(out[:5], want, size)
        assert bool((out[5:] == 3.0).all()) and bool((wide[:, :8 * 64] == 3.0).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_queries_in_a_wider_projection(fp8):
    new, total = [40, 3], [300, 200]
    case, dense = _case(new, total, 8, 2, 64, 64, fp8)
    want, size = _oracle(case["q"], dense, new, total, None, 0, 64 ** -0.5)
    for pad in (8, 5):                                       # rows at 16-byte addresses, and not
        wide = torch.full((43, 8 * 64 + pad), float("nan"), dtype=torch.bfloat16, device=DEV)
        wide[:, :8 * 64] = case["q"].flatten(1)
        case["q"] = wide[:, :8 * 64].view(43, 8, 64)
        _close(_run(case, new), want, size)


def test_hidden_keys_may_be_nan_and_a_seen_one_says_so():
    new, total = [4], [260]
    for fp8 in (False, True):
        case, dense = _case(new, total, 4, 2, 64, 64, fp8)
        page = int(case["table"][0, 4])
        if fp8:
            case["ks"][page, :, 3] = 255                     # the last token's key: earlier queries do not see it
        else:
            case["k"][page, 3] = float("nan")
        got = _run(case, new)
        want, size = _oracle(case["q"], dense, new, total, None, 0, 64 ** -0.5)
        _close(got[:3], want[:3], size[:3])
        assert torch.isnan(got[3]).all()


def test_a_step_is_captured_and_replayed_with_other_lengths():
    total = [500, 130, 64]
    case, dense = _case([1, 1, 1], total, 8, 2, 128, 64, True, dirty=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call = lambda: C.cache_attention(case["q"], case["k"], case["v"], case["table"], case["lens"], k_scale=case["ks"], v_scale=case["vs"], splits=3)
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                       # two graphs, replayed in turn: neither's scratch is the other's
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for lens in (total, [77, 130, 1], [0, 5, 64]):
        case["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        part = [[t[:n] for t in x] for x, n in zip(dense, lens)]
        want, size = _oracle(case["q"], part, [1, 1, 1], lens, None, 0, 128 ** -0.5)
        for _, out in graphs:
            _close(out, want, size)
    check_status()


def test_streams_of_their_own_do_not_disturb_each_other():
    new, total = [37, 2], [900, 1500]
    jobs = []
    for i in range(4):
        case, dense = _case(new, total, 8, 2, 128, 64, i % 2 == 1, seed=i)
        jobs.append((case, _oracle(case["q"], dense, new, total, None, 0, 128 ** -0.5), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for case, _, s in jobs:
            with torch.cuda.stream(s):
                outs.append(_run(case, new, splits=3))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        _close(o, *jobs[i % 4][1])


@pytest.mark.parametrize("fp8", [False, True])
def test_the_same_call_gives_the_same_bits(fp8):
    new, total = [50, 2, 1], [900, 1500, 2000]
    case, _ = _case(new, total, 8, 2, 128, 64, fp8)
    first = _run(case, new)
    assert all(torch.equal(first, _run(case, new)) for _ in range(5))


def test_offsets_past_32_bits():
    """Pages at the end of a pool of over 2^31 numbers."""
    hk, d, block = 8, 128, 64
    blocks = (1 << 31) // (block * hk * d) + 40
    total, new = [300, 70], [2, 1]
    small, dense = _case(new, total, 16, hk, d, block, False, dirty=False)
    want = _run(small, new)
    pool = torch.zeros(blocks, block, hk, d, dtype=torch.bfloat16, device=DEV)
    n = small["k"].shape[0]
    table = torch.where(small["table"] >= 0, small["table"] + blocks - n, small["table"])
    pool[-n:] = small["k"]
    got = C.cache_attention(small["q"], pool, pool, table, small["lens"], small["cu"], 2)
    assert torch.equal(got, C.cache_attention(small["q"], small["k"], small["k"], small["table"], small["lens"], small["cu"], 2))
    del pool
    codes, scale = torch.zeros(blocks, block, hk, d, dtype=torch.uint8, device=DEV).view(F8), torch.zeros(blocks, hk, block, dtype=torch.uint8, device=DEV)
    rows = torch.randn(5, hk * d, device=DEV).to(torch.bfloat16)
    slots = torch.tensor([blocks * block - 1, 3, blocks * block - 70, -1, blocks * block - 64], dtype=torch.int32, device=DEV)
    C.kv_cache_write_fp8(rows, rows, codes, codes, scale, scale, slots)
    back, _ = C.kv_cache_read_fp8(codes, codes, scale, scale, slots)
    exact = ref._fp8_values(*ref.fp8_rows(rows.cpu().view(5, hk, d))).view(5, -1).to(torch.bfloat16)
    exact[3] = 0
    assert torch.equal(back.cpu(), exact)
    check_status()
    assert want.shape == got.shape


@pytest.mark.parametrize("bad", ["table", "length", "negative", "cu"])
def test_bad_tables_and_lengths_are_reported(bad):
    new, total = [2, 1], [200, 100]
    case, _ = _case(new, total, 4, 2, 64, 64, False, dirty=False)
    if bad == "table":
        case["table"][0, 1] = 10 ** 6
    elif bad == "length":
        case["lens"][0] = 10 ** 6
    elif bad == "negative":
        case["lens"][1] = -5
    else:
        case["cu"][2] = 9
    _run(case, new)
    with pytest.raises(KernelStatusError):
        check_status()


def test_refusals():
    new, total = [2], [20]
    case, _ = _case(new, total, 4, 2, 64, 16, False)
    call = lambda **kw: C.cache_attention(**{**dict(q=case["q"], k_cache=case["k"], v_cache=case["v"], block_table=case["table"], seq_lens=case["lens"],
                                                    cu_q=case["cu"], max_q=2), **kw})
    call()
    scale = torch.zeros(case["k"].shape[0], 2, 16, dtype=torch.uint8, device=DEV)
    for kw in (dict(q=case["q"].float()), dict(q=case["q"][:, :3]), dict(k_cache=case["k"].float()), dict(k_cache=case["k"][:, :8]),
               dict(k_cache=case["k"][:, ::2]), dict(k_scale=scale), dict(k_scale=scale, v_scale=scale), dict(block_table=case["table"].long()),
               dict(seq_lens=case["lens"].repeat(2)), dict(cu_q=case["cu"][:1]), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf),
               dict(first_tokens=-1), dict(out=case["q"].float()), dict(out=case["q"].transpose(0, 1)), dict(q=case["q"].cpu().to(DEV).expand(2, 4, 64)[:, :, :32]),
               dict(seq_lens=case["lens"].cpu())):
        with pytest.raises(RuntimeError):
            call(**kw)
    for window in (0, -3):
        with pytest.raises(ValueError):
            call(window=window)
    pages = _empty(2, 16, 2, 64)
    k = torch.zeros(3, 128, dtype=torch.bfloat16, device=DEV)
    slots = torch.zeros(3, dtype=torch.int32, device=DEV)
    C.kv_cache_write_fp8(k, k, *pages, slots)
    for args in ((k.float(), k, *pages, slots), (k[:, :64], k[:, :64], *pages, slots), (k, k, *pages, slots[:2]), (k, k, *pages, slots.long()),
                 (k, k, pages[0].view(torch.uint8), *pages[1:], slots), (k, k, *pages[:2], pages[2][:, :1], pages[3], slots), (k, k[:2], *pages, slots)):
        with pytest.raises(RuntimeError):
            C.kv_cache_write_fp8(*args)
    with pytest.raises(RuntimeError):
        C.kv_cache_read_fp8(*pages, slots.float())
    check_status()


def test_nothing_to_do():
    case, _ = _case([2], [20], 4, 2, 64, 16, False)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert C.cache_attention(case["q"][:0], case["k"], case["v"], case["table"], case["lens"], torch.zeros(2, dtype=torch.int32, device=DEV), 0).shape == (0, 4, 64)
    assert not C.cache_attention(case["q"], case["k"], case["v"], case["table"][:0], none, torch.zeros(1, dtype=torch.int32, device=DEV), 0).any()
    pages = _empty(2, 16, 2, 64)
    C.kv_cache_write_fp8(*(torch.zeros(0, 128, dtype=torch.bfloat16, device=DEV),) * 2, *pages, none)
    assert C.kv_cache_read_fp8(*pages, none)[0].shape == (0, 128)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new", [[3, 2], [70, 90]])
def test_rows_in_front_of_the_first_sequence(fp8, new):
    total = [400, 150]
    case, dense = _case(new, total, 8, 2, 64, 64, fp8)
    want, size = _oracle(case["q"], dense, new, total, None, 0, 64 ** -0.5)
    case["q"] = torch.cat([torch.full_like(case["q"][:2], float("nan")), case["q"]])
    case["cu"] += 2
    torch.full((64, 8, 64), float("nan"), dtype=torch.bfloat16, device=DEV)                   # what the result may be given to lie in
    got = _run(case, new)
    check_status()
    assert not got[:2].any()
    _close(got[2:], want, size)
    out = torch.full_like(case["q"], 3.0)
    _run(case, new, out=out)
    assert torch.equal(out[2:], got[2:]) and torch.equal(out[:2], torch.full_like(out[:2], 3.0))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hk,cu", [(4, 2, True), (4, 2, False), (96, 1, False)])
def test_more_sequences_than_one_launch_holds(fp8, hq, hk, cu):
    """1300 sequences of 0 to 70 tokens, one new token each or (with cu_q) none to two; 96 query heads over one key head."""
    n = 1300
    g = torch.Generator().manual_seed(3)
    new = torch.randint(0, 3, (n,), generator=g).tolist() if cu else [1] * n
    total = [max(a, m) for a, m in zip(torch.randint(0, 71, (n,), generator=g).tolist(), new)] if cu else torch.randint(0, 71, (n,), generator=g).tolist()
    case, dense = _case(new, total, hq, hk, 64, 16, fp8, dirty=False)
    want, size = _oracle(case["q"], dense, new, total, None, 0, 64 ** -0.5)
    if not cu:
        case["cu"] = None
    got = _run(case, new)
    check_status()
    _close(got, want, size)


def test_queries_that_share_their_memory():
    new, total = [5], [300]
    case, dense = _case(new, total, 4, 2, 64, 64, False)
    one = case["q"][:1].clone()
    case["q"] = one.expand(5, 4, 64)
    got = _run(case, new)
    case["q"] = one.repeat(5, 1, 1)
    assert torch.equal(got, _run(case, new))
    check_status()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window,first", [(None, 0), (5000, 200)])
@pytest.mark.parametrize("new,total,cu", [([1], [20000], True), ([1, 1, 1], [9000, 0, 14001], False), ([4, 2], [4, 12345], True)])
def test_few_tokens_of_long_sequences(new, total, cu, window, first, fp8):
    case, dense = _case(new, total, 32, 8, 128, 64, fp8, window=window, first=first)
    want, size = _oracle(case["q"], dense, new, total, window, first, 128 ** -0.5)
    if not cu:
        case["cu"] = None
    got = _run(case, new, window=window, first_tokens=first)
    check_status()
    _close(got, want, size)
