"""Attention over 8-bit pages where sizes are unusual: value rows that differ much, tables far wider than what is seen, entries and lengths
that are out of range.  Against plain math in 64 bits."""
import pytest
import torch

from pisceslx_b200.ops import cache as C
from pisceslx_b200.ops import KernelStatusError, check_status
from pisceslx_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _powers(kind, n, new, g):
    """A power of two for each value row, and what is added to each key's scores (natural units)."""
    power, score = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    if kind == "rising":                              # each tile's largest is far above the ones before it
        power = torch.linspace(-40, 30, n).round().double()
    elif kind == "falling":
        power = torch.linspace(30, -40, n).round().double()
    elif kind == "hidden":                            # the last token's row: hidden from all queries but the last, and far off for that one
        power[-1], score[-1] = 30, -60.0
    elif kind == "unlikely":                          # a large row that carries no weight, after others of the usual size
        power[n // 2], score[n // 2] = 30, -60.0
    elif kind == "sink":                              # the first token has nearly all the weight and a tiny row; 2^-31 of the weight meets rows 2^30 larger
        power[0], score[0] = -30, 21.5
    elif kind == "random":
        power = torch.randint(-30, 31, (n,), generator=g).double()
    elif kind == "extremes":                          # sums in 32 bits hold rows down to 2^-100 of the largest
        power = torch.full((n,), -60.0, dtype=torch.float64)
        power[n // 3], score[n // 3] = 40, -80.0
    return power, score


def _case(kind, new, total, hq, hk, d, block, seed=0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in total]
    order = torch.randperm(sum(need) + 1, generator=g).tolist()
    table = torch.full((len(total), max(need)), -1, dtype=torch.int32)
    pages = [torch.zeros(len(order), block, hk, d, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.zeros(len(order), hk, block, dtype=torch.uint8) for _ in range(2)]
    dense = []
    for b, n in enumerate(total):
        power, score = _powers(kind, n, new[b], g)
        k = torch.randn(n, hk, d, generator=g) * 0.5
        k[:, :, 0] = score[:, None].float() / 8.0                       # every query has 8 sqrt(d) there
        v = torch.randn(n, hk, d, generator=g).double() * torch.exp2(power)[:, None, None]
        rows = []
        for x, pool, scale in zip((k.to(torch.bfloat16), v.to(torch.bfloat16)), pages, scales):
            codes, byte = ref.fp8_rows(x)
            for p in range(need[b]):
                page = order[sum(need[:b]) + p]
                table[b, p] = page
                part = slice(p * block, min((p + 1) * block, n))
                m = part.stop - part.start
                pool[page, :m] = codes.view(torch.uint8)[part]
                scale[page, :, :m] = byte[part].t()
            rows.append(ref._fp8_values(codes, byte))
        dense.append(rows)
    q = torch.randn(sum(new), hq, d, generator=g).to(torch.bfloat16)
    q[:, :, 0] = 8.0 * d ** 0.5
    f8 = lambda t: t.to(DEV).view(torch.float8_e4m3fn)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    args = (q.to(DEV), f8(pages[0]), f8(pages[1]), table.to(DEV), torch.tensor(total, dtype=torch.int32, device=DEV), cu.to(DEV), max(new))
    return args, dict(k_scale=scales[0].to(DEV), v_scale=scales[1].to(DEV)), dense


def _oracle(q, dense, new, window, first):
    outs, sizes, at = [], [], 0
    for (k, v), m in zip(dense, new):
        n, hk, d = k.shape
        k, v = (x.double().to(DEV).repeat_interleave(q.shape[1] // hk, 1) for x in (k, v))
        i, j = torch.arange(n - m, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        ok = j <= i
        if window is not None:
            ok &= (i - j < window) | (j < first)
        sc = (torch.einsum("mhd,nhd->hmn", q[at:at + m].double(), k) * d ** -0.5).masked_fill(~ok, float("-inf"))
        w = torch.softmax(sc, -1)
        outs.append(torch.einsum("hmn,nhd->mhd", w, v))
        sizes.append(torch.einsum("hmn,nhd->mhd", w, v.abs()))
        at += m
    return torch.cat(outs), torch.cat(sizes)


def _close(got, want, size):
    """Weights are rounded to 8 bits at worst (2^-8 of each), the result too (2^-8 of it).  The rest is within 2^-10 of what the weights
    make of the values: 2^x to 1e-4, and fp16 weights, which are off by 2^-29 of the largest row beside others within 2^7 of it, 2^-22
    of what counts most for each key: 2^-12 where 1000 keys are all rounded alike (2100 rounded at random: 2^-16)."""
    top = size.amax(-1, keepdim=True)                 # codes of one row differ in size: what a weight is off by is relative to the row
    bad = (got.double() - want).abs() > (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -12 * top + 2.0 ** -8 * want.abs()
    assert torch.isfinite(got).all() and not bad.any(), (int(bad.sum()), bad.numel(), float(((got.double() - want).abs() / top).max()))


KINDS = ["rising", "falling", "hidden", "unlikely", "sink", "random", "extremes"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hk,new", [(8, 2, 1), (8, 1, 1), (8, 2, 4), (8, 2, 7), (8, 2, 16), (8, 2, 20)])
@pytest.mark.parametrize("d,block", [(128, 64), (64, 16)])
def test_value_rows_of_many_sizes(kind, hq, hk, new, d, block):
    """4 to 64 rows of queries beside one another (and 80, which another kernel takes)."""
    news, total = [new, 1, new], [1000, 130, max(new, 300)]
    args, scales, dense = _case(kind, news, total, hq, hk, d, block, seed=new)
    got = C.cache_attention(*args, **scales)
    check_status()
    _close(got, *_oracle(args[0], dense, news, None, 0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 3, 12])
def test_long_sequences_in_pieces(kind, new):
    """Enough tiles that every piece of the line has several, and sequences are cut."""
    news, total = [new] * 24, [2100] * 24
    args, scales, dense = _case(kind, news, total, 16, 4, 128, 64, seed=new)
    got = C.cache_attention(*args, **scales)
    check_status()
    _close(got, *_oracle(args[0], dense, news, None, 0))


@pytest.mark.parametrize("kind", ["unlikely", "hidden", "random", "falling"])
@pytest.mark.parametrize("window,first", [(100, 0), (260, 130), (1, 3)])
@pytest.mark.parametrize("new", [1, 9])
def test_large_rows_behind_a_window(kind, window, first, new):
    news, total = [new, new], [900, 515]
    args, scales, dense = _case(kind, news, total, 8, 2, 128, 64, seed=window)
    got = C.cache_attention(*args, window=window, first_tokens=first, **scales)
    check_status()
    _close(got, *_oracle(args[0], dense, news, window, first))


def test_the_number_of_rows_does_not_change_what_a_token_gets():
    """64 rows and 68 rows run in kernels of two kinds: the tokens that both calls have get the same but for roundings."""
    (q, *rest), scales, dense = _case("hidden", [17], [800], 8, 2, 128, 64)
    table, lens = rest[2], rest[3]
    all_rows = C.cache_attention(q, *rest[:4], torch.tensor([0, 17], dtype=torch.int32, device=DEV), 17, **scales)
    few = C.cache_attention(q[1:].contiguous(), rest[0], rest[1], table, lens, torch.tensor([0, 16], dtype=torch.int32, device=DEV), 16, **scales)
    want, size = _oracle(q, dense, [17], None, 0)
    _close(all_rows, want, size)
    _close(few, want[1:], size[1:])


def _wide_table(args, width):
    """The same call with a table of as many entries as a long stream has: those in front were given back, those behind are not used."""
    table = torch.full((args[3].shape[0], width), -1, dtype=torch.int32, device=DEV)
    table[:, :args[3].shape[1]] = args[3]
    return args[:3] + (table,) + args[4:]


@pytest.mark.parametrize("window,first", [(100, 0), (300, 4), (700, 200), (129, 128), (1, 0), (2000, 700)])
def test_scratch_of_a_windowed_portion_follows_the_window(window, first):
    news, total = [90, 33], [1900, 640]
    args, scales, dense = _case("even", news, total, 8, 2, 128, 64, seed=window)
    want, size = _oracle(args[0], dense, news, window, first)
    _close(C.cache_attention(*args, window=window, first_tokens=first, **scales), want, size)
    args = _wide_table(args, 40000)                                              # 2560000 tokens: 2.6 GB a sequence in bf16
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = C.cache_attention(*args, window=window, first_tokens=first, **scales)
    check_status()
    _close(got, want, size)
    rows = -(-first // 128) * 128 + window + 90 + 256
    # keys and values of what can be seen, and up to 32 ranges of sums in 32 bits
    assert torch.cuda.max_memory_allocated() - before < 2 * (rows * 2 * 128 * 4) + 32 * 123 * 8 * 130 * 4 + (1 << 20)


def test_widened_pages_of_a_batch_in_turns():
    """Tables of 131072 tokens: two sequences of 8 heads of 128 are widened at a time."""
    news, total = [40, 20, 33, 1, 17], [700, 300, 33, 260, 129]
    args, scales, dense = _case("even", news, total, 32, 8, 128, 64)
    want, size = _oracle(args[0], dense, news, None, 0)
    _close(C.cache_attention(*args, **scales), want, size)
    wide = _wide_table(args, 2048)
    got = C.cache_attention(*wide, **scales)
    check_status()
    _close(got, want, size)
    out = torch.full_like(args[0], 3.0)
    C.cache_attention(*wide, out=out, splits=2, **scales)
    check_status()
    _close(out, want, size)


@pytest.mark.parametrize("bad", ["table", "length", "negative", "queries", "backwards"])
@pytest.mark.parametrize("new", [[2, 1], [16, 1], [90, 2]])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window", [None, 150])
def test_what_is_out_of_range_is_reported_and_disturbs_no_other_sequence(bad, new, fp8, window):
    """Bad entries in the middle of three sequences, in each of the kernels."""
    news, total = [new[0], new[0], new[1]], [300, 200, 130]
    (q, k, v, table, lens, cu, max_q), scales, dense = _case("even", news, total, 8, 2, 64, 64)
    want, size = _oracle(q, dense, news, window, 0)
    if not fp8:
        k, v = (torch.ldexp(x.float(), (s.transpose(1, 2).int() - 127).unsqueeze(-1)).to(torch.bfloat16) for x, s in
                ((k, scales["k_scale"]), (v, scales["v_scale"])))
        scales = {}
    if bad == "table":
        table[1, 1:4] = torch.tensor([10 ** 6, -1, 2 ** 31 - 1], dtype=torch.int32)
    elif bad == "length":
        lens[1] = 2 ** 31 - 1
    elif bad == "negative":
        lens[1] = -2 ** 31
    elif bad == "queries":
        max_q = new[0] + new[1]
        cu[1:] += torch.tensor([0, 2 ** 30, 2 ** 30], dtype=torch.int32, device=DEV)
    else:
        cu[2] = 0
    got = C.cache_attention(q, k, v, table, lens, cu, max_q, window=window, **scales)
    with pytest.raises(KernelStatusError):
        check_status()
    _close(got[:new[0]], want[:new[0]], size[:new[0]])
    if bad in ("table", "length", "negative"):
        _close(got[2 * new[0]:], want[2 * new[0]:], size[2 * new[0]:])
    check_status()


@pytest.mark.parametrize("news", [[3, 1], [40, 7]])
def test_the_largest_number_of_new_tokens_need_not_be_given(news):
    args, scales, dense = _case("even", news, [200, 90], 8, 2, 64, 64)
    got = C.cache_attention(*args[:6], **scales)
    check_status()
    _close(got, *_oracle(args[0], dense, news, None, 0))
    C.cache_attention(*args[:6], max(news) - 1, **scales)
    with pytest.raises(KernelStatusError):
        check_status()
