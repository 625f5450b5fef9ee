"""Performance cases of the operators around a paged cache of 8-bit keys and values.

Three operators of ``ops.cache``, each through the call that a serving program makes:

* ``write``   ``kv_cache_write_fp8``: new keys and values become e4m3 codes in their pages, with one power-of-two scale for each
              token and head;
* ``read``    ``kv_cache_read_fp8``: cached tokens, wherever their pages lie, as bf16 rows;
* ``attend``  ``cache_attention``: the new tokens of every sequence over what the pages hold, in 8 bits or in bf16, causal, with
              an optional window and a few first tokens that stay visible.  One new token per sequence is a decode step.

Heads are those of the repository's presets; pages hold 64 tokens, the engine's default, and lie in no order."""
from __future__ import annotations

import math
import random
from typing import Any, Dict, List, Tuple

import torch

own = False

DEV = "cuda"
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
PAGE = 64
E4M3_MAX = 448.0


def listed() -> List[Dict[str, Any]]:
    wide = dict(hq=32, hk=8, d=128)
    narrow = dict(hq=16, hk=4, d=64)
    return [
        # one conversation's next token goes into the cache of one layer
        dict(name="write_one", kind="write", tokens=1, hk=8, d=128),
        # the next tokens of the serving benchmark's batch, small heads
        dict(name="write_batch", kind="write", tokens=64, hk=4, d=64),
        # a document-sized prompt, not a whole number of pages
        dict(name="write_prompt", kind="write", tokens=8191, hk=8, d=128),
        # a short prefix is taken out of the cache
        dict(name="read_short", kind="read", tokens=131, hk=4, d=64),
        # a long document is taken out of the cache
        dict(name="read_long", kind="read", tokens=32768, hk=8, d=128),
        # interactive decoding of one conversation over bf16 pages
        dict(name="decode_one", kind="attend", batch=1, new=1, context=2048, window=0, first=0, fp8=False, **wide),
        # the serving benchmark's batch over 8-bit pages; contexts between half and all of 4096 tokens
        dict(name="decode_batch_fp8", kind="attend", batch=64, new=1, context=4096, window=0, first=0, fp8=True, **wide),
        # streams far past their window, whose first tokens stay visible
        dict(name="decode_stream", kind="attend", batch=16, new=1, context=30011, window=4096, first=4, fp8=False, **wide),
        # drafts of five tokens are verified over 8-bit pages
        dict(name="verify_fp8", kind="attend", batch=8, new=5, context=8192, window=0, first=0, fp8=True, **wide),
        # short turns of several conversations, of lengths of their own, small heads, windowed 8-bit pages
        dict(name="turns_fp8", kind="attend", batch=5, new=301, context=2777, window=1024, first=16, fp8=True, **narrow),
        # one portion of a long prompt over bf16 pages
        dict(name="portion", kind="attend", batch=1, new=512, context=16384, window=0, first=0, fp8=False, **wide),
        # a large portion of a long document over 8-bit pages
        dict(name="document_fp8", kind="attend", batch=1, new=4096, context=32768, window=0, first=0, fp8=True, **wide),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> Dict[str, Any]:
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
    hq, hk, d = rng.choice([(32, 8, 128), (16, 4, 64), (64, 8, 128), (16, 4, 128), (8, 2, 64), (16, 16, 64)])
    if kind != "attend":
        return dict(kind=kind, tokens=_log(rng, 1, 8191 if kind == "write" else 32768), hk=min(hk, 8), d=d)
    form = rng.choice(["decode", "few", "portion"])
    if form == "decode":
        batch, new = _log(rng, 1, 64), 1
    elif form == "few":
        batch, new = _log(rng, 1, 32), rng.randint(2, 16)
    else:
        batch, new = rng.randint(1, 4), _log(rng, 17, 2048)
    context = new + _log(rng, 1, min(32768, 262144 // batch) - new)
    if hk > 8:                                     # no heads shared: eight times the wide model's keys per query
        context = new + (context - new) // 2
    context = max(new, min(context, int(5e11 / (batch * new * hq * d))))          # no more than the largest listed case
    window = rng.choice([0, 0, _log(rng, 64, 8192)])
    return dict(kind=kind, batch=batch, new=new, context=context, window=window, first=rng.choice([0, 4, 64, 100]) if window else 0,
                fp8=rng.random() < 0.5, hq=hq, hk=hk, d=d)


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _rows(gen: torch.Generator, n: int, heads: int, d: int, key: bool) -> torch.Tensor:
    """Keys or values [n, heads, d] fp32 as a trained layer has them: a few channels of every key head are much larger."""
    x = torch.randn(n, heads, d, device=DEV, generator=gen)
    if key:
        x = x * torch.exp(torch.randn(heads, d, device=DEV, generator=gen) * 0.7)
    return x


def _codes(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., d] -> e4m3 codes and exponent bytes [...]: the smallest power of two at which the largest number fits."""
    top = x.float().abs().amax(-1)
    m, e = torch.frexp(top)                        # top = m 2^e, m in [1/2, 1); 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).int()
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
    y = torch.ldexp(x.float(), -e.unsqueeze(-1))
    return y.to(F8), (e + 127).to(torch.uint8)


def _lengths(case: Dict[str, Any]) -> Tuple[List[int], List[int]]:
    """New tokens and all tokens of each sequence: the first has the case's, the others between half and all of them."""
    rng = random.Random(case["batch"])
    some = lambda n: rng.randint((n + 1) // 2, n)
    new = [case["new"] if i == 0 or case["new"] <= 16 else some(case["new"]) for i in range(case["batch"])]
    return new, [case["context"] if i == 0 else max(n, some(case["context"])) for i, n in enumerate(new)]


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    hk, d = case["hk"], case["d"]
    if case["kind"] != "attend":
        T = case["tokens"]
        pages = -(-T // PAGE) + 3
        ids = torch.randperm(pages, device=DEV, generator=gen)
        at = torch.arange(T, device=DEV)
        slots = (ids[at // PAGE] * PAGE + at % PAGE).int()
        if case["kind"] == "write":                # keys and values lie next to each other in the projection
            kv = torch.cat([_rows(gen, T, hk, d, True).view(T, -1), _rows(gen, T, hk, d, False).view(T, -1)], 1).to(BF16)
            codes = lambda: torch.zeros(pages, PAGE, hk, d, device=DEV).to(F8)
            scales = lambda: torch.zeros(pages, hk, PAGE, dtype=torch.uint8, device=DEV)
            return dict(case=case, k=kv[:, :hk * d], v=kv[:, hk * d:], slots=slots,
                        pages=[codes(), codes(), scales(), scales()])
        kc, ks = _codes(_rows(gen, pages * PAGE, hk, d, True).view(pages, PAGE, hk, d))
        vc, vs = _codes(_rows(gen, pages * PAGE, hk, d, False).view(pages, PAGE, hk, d))
        return dict(case=case, slots=slots, pages=[kc, vc, ks.transpose(1, 2).contiguous(), vs.transpose(1, 2).contiguous()])
    new, total = _lengths(case)
    need = [-(-n // PAGE) for n in total]
    pages = sum(need) + 1
    ids = torch.randperm(pages, device=DEV, generator=gen).int()
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    k, v = (torch.empty(pages, PAGE, hk, d, dtype=F8 if case["fp8"] else BF16, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(pages, hk, PAGE, dtype=torch.uint8, device=DEV) if case["fp8"] else None for _ in range(2))
    widths = torch.exp(torch.randn(hk, d, device=DEV, generator=gen) * 0.7)
    for lo in range(0, pages, 256):                # in portions: the numbers in 32 bits take four times the codes' room
        n = min(256, pages - lo)
        for pool, scale, w in ((k, ks, widths), (v, vs, None)):
            x = torch.randn(n, PAGE, hk, d, device=DEV, generator=gen)
            x = x * w if w is not None else x
            if scale is None:
                pool[lo:lo + n] = x.to(BF16)
            else:
                code, e = _codes(x)
                pool[lo:lo + n].view(torch.uint8).copy_(code.view(torch.uint8))
                scale[lo:lo + n] = e.transpose(1, 2)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], case["hq"], d, device=DEV, generator=gen).to(BF16)
    return dict(case=case, q=q, k=k, v=v, ks=ks, vs=vs, table=table, new=new, total=total, cuts=cu, max_new=max(new),
                lens=torch.tensor(total, dtype=torch.int32, device=DEV),
                cu=torch.tensor(cu, dtype=torch.int32, device=DEV) if case["new"] > 1 else None)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _take(pool: torch.Tensor, scale, page: torch.Tensor, offset: torch.Tensor) -> torch.Tensor:
    """Cached rows [..., heads, d] in 32 bits at pages and places within them."""
    x = pool.view(torch.uint8)[page, offset].view(F8).float() if scale is not None else pool[page, offset].float()
    if scale is not None:
        x = torch.ldexp(x, (scale[page, :, offset].int() - 127).unsqueeze(-1))
    return x


def _plain_write(s: Dict[str, Any]):
    k_pages, v_pages, k_scale, v_scale = s["pages"]
    hk, d = s["case"]["hk"], s["case"]["d"]
    page, offset = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    for x, pool, scale in ((s["k"], k_pages, k_scale), (s["v"], v_pages, v_scale)):
        code, e = _codes(x.reshape(-1, hk, d))
        pool.view(torch.uint8)[page, offset] = code.view(torch.uint8)
        scale[page, :, offset] = e
    return k_pages, v_pages, k_scale, v_scale


def _plain_read(s: Dict[str, Any]):
    k_pages, v_pages, k_scale, v_scale = s["pages"]
    page, offset = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    return tuple(_take(p, e, page, offset).flatten(1).to(BF16) for p, e in ((k_pages, k_scale), (v_pages, v_scale)))


def _softmax_products(q, k, v, ok, scale):
    """q [b, m, hk, g, d], k and v [b, n, hk, d], ok [b, m, n] -> [b, m, hk, g, d]."""
    sc = torch.einsum("bmhgd,bnhd->bhgmn", q, k).mul_(scale).masked_fill_(~ok[:, None, None], float("-inf"))
    w = sc.sub_(sc.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = w.sum(-1)
    o = torch.einsum("bhgmn,bnhd->bmhgd", w, v)
    return o / total.permute(0, 3, 1, 2).unsqueeze(-1).clamp_min(1e-38)


def _plain_attend(s: Dict[str, Any]) -> torch.Tensor:
    c, q, table = s["case"], s["q"], s["table"]
    hq, hk, d, window, first = c["hq"], c["hk"], c["d"], c["window"], c["first"]
    out = torch.empty_like(q)

    def visible(b0: int, b1: int, m: int):
        """Positions of the keys that sequences b0 .. b1 - 1 see, and of their last m tokens; padded to one count."""
        n = s["lens"][b0:b1].long()[:, None]
        starts = [max(0, t - k - window + 1) if window else 0 for t, k in zip(s["total"][b0:b1], s["new"][b0:b1])]
        lo = torch.tensor(starts, device=DEV)[:, None]
        ahead = lo.clamp_max(first)
        count = max(min(first, a) + t - a for a, t in zip(starts, s["total"][b0:b1]))
        j = torch.arange(count, device=DEV)[None]
        pos = torch.where(j < ahead, j, j - ahead + lo)
        return torch.where(pos < n, pos, torch.full_like(pos, -1)), n - m + torch.arange(m, device=DEV)[None]

    def keys(b0: int, b1: int, pos: torch.Tensor, heads: slice):
        at = pos.clamp_min(0)
        page = table[b0:b1].long().gather(1, at // PAGE)
        sl = lambda t, dim: None if t is None else t.narrow(dim, heads.start, heads.stop - heads.start)
        return (_take(sl(s["k"], 2), sl(s["ks"], 1), page, at % PAGE), _take(sl(s["v"], 2), sl(s["vs"], 1), page, at % PAGE))

    def mask(pos: torch.Tensor, mine: torch.Tensor) -> torch.Tensor:
        p, m = pos[:, None, :], mine[:, :, None]
        ok = (p >= 0) & (p <= m)
        return ok & ((p > m - window) | (p < first)) if window else ok

    step = 1 if s["max_new"] > 16 else max(1, (1 << 18) // max(s["total"]))
    for b0 in range(0, len(s["new"]), step):
        b1 = min(len(s["new"]), b0 + step)
        m = s["new"][b0]
        pos, mine = visible(b0, b1, m)
        ok = mask(pos, mine)
        rows = q[s["cuts"][b0]:s["cuts"][b1]].view(b1 - b0, m, hk, hq // hk, d)
        dst = out[s["cuts"][b0]:s["cuts"][b1]].view(b1 - b0, m, hk, hq // hk, d)
        at_once = hk if m <= 16 else max(1, min(hk, (1 << 29) // (m * (hq // hk) * pos.shape[1])))
        for h in range(0, hk, at_once):
            hs = slice(h, min(hk, h + at_once))
            k, v = keys(b0, b1, pos, hs)
            dst[:, :, hs] = _softmax_products(rows[:, :, hs].float(), k, v, ok, d ** -0.5).to(BF16)
    return out


def run(state: Dict[str, Any]):
    case = state["case"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[case["kind"]](state)
    from pisceslx_b200.ops import cache as C
    if case["kind"] == "write":
        C.kv_cache_write_fp8(state["k"], state["v"], *state["pages"], state["slots"])
        return tuple(state["pages"])
    if case["kind"] == "read":
        return C.kv_cache_read_fp8(*state["pages"], state["slots"])
    return C.cache_attention(state["q"], state["k"], state["v"], state["table"], state["lens"], state["cu"], state["max_new"],
                             window=case["window"] or None, first_tokens=case["first"], k_scale=state["ks"], v_scale=state["vs"])


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ------------------------------------------------------------------------------------------------
def _visible_pairs(new: int, total: int, window: int, first: int) -> Tuple[int, int]:
    """(query, key) pairs of one sequence, and keys that any of its new tokens sees."""
    pairs = 0
    for p in (range(total - new, total) if window else ()):
        lo = max(0, p - window + 1)
        pairs += p + 1 - lo + min(first, lo)
    if not window:
        return new * total - new * (new - 1) // 2, total
    lo = max(0, total - new - window + 1)
    return pairs, total - lo + min(first, lo)


def work(case: Dict[str, Any]) -> Dict[str, float]:
    hk, d = case["hk"], case["d"]
    if case["kind"] != "attend":
        row = 2 * hk * d
        return {"bytes": float(case["tokens"] * (row * 3 + 2 * hk + 4)), "flops": float(2 * case["tokens"] * row)}
    new, total = _lengths(case)
    seen = [_visible_pairs(n, t, case["window"], case["first"]) for n, t in zip(new, total)]
    key = 2 * hk * (d + 1 if case["fp8"] else 2 * d)
    return {"bytes": float(sum(new) * case["hq"] * d * 4 + sum(k for _, k in seen) * key),
            "flops": 4.0 * d * case["hq"] * sum(p for p, _ in seen)}


def _exact_codes(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Values of the codes and exponents, by their definition, in 64 bits: codes are multiples of 2^(floor(log2 |y|) - 3), and of
    2^-9 below 2^-6; halves go to the even one."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -127.0)
    for c in range(-126, 128):
        e = torch.where(top > E4M3_MAX * 2.0 ** (c - 1), torch.full_like(e, float(c)), e)
    y = x * torch.pow(2.0, -e)
    a = y.abs()
    step = torch.full_like(a, 2.0 ** -9)
    for c in range(-5, 9):
        step = torch.where(a >= 2.0 ** c, torch.full_like(a, 2.0 ** (c - 3)), step)
    n = a / step
    low = n.floor()
    up = (n - low > 0.5) | ((n - low == 0.5) & (low % 2 == 1))
    return torch.sign(y) * (low + up.double()) * step, e.squeeze(-1)


def exact(case: Dict[str, Any], seed: int):
    s = prepare(case, seed)
    hk, d = case["hk"], case["d"]
    value = lambda pool, scale: pool.double() * torch.pow(2.0, scale.double() - 127).transpose(1, 2).unsqueeze(-1)
    if case["kind"] == "write":
        out = []
        at = s["slots"].long()
        for x in (s["k"], s["v"]):
            code, e = _exact_codes(x.reshape(-1, hk, d))
            pool = torch.zeros(s["pages"][0].shape, dtype=torch.float64, device=DEV)
            pool.view(-1, hk, d)[at] = code
            scale = torch.zeros(pool.shape[0], PAGE, hk, dtype=torch.uint8, device=DEV)
            scale.view(-1, hk)[at] = (e + 127).to(torch.uint8)
            out.append((pool, scale.transpose(1, 2).contiguous()))
        return out[0][0], out[1][0], out[0][1], out[1][1]
    if case["kind"] == "read":
        kc, vc, ks, vs = s["pages"]
        return tuple(value(p, e).reshape(-1, hk * d)[s["slots"].long()] for p, e in ((kc, ks), (vc, vs)))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    group = case["hq"] // hk
    for b, (new, total) in enumerate(zip(s["new"], s["total"])):
        pages = s["table"][b, :-(-total // PAGE)].long()
        far = torch.arange(total - new, total, device=DEV)[:, None] - torch.arange(total, device=DEV)[None]
        hidden = far < 0
        if case["window"]:
            hidden |= (far >= case["window"]) & (torch.arange(total, device=DEV)[None] >= case["first"])
        for h in range(hk):
            heads = slice(h * group, (h + 1) * group)
            k, v = ((value(p[pages, :, h:h + 1], e[pages, h:h + 1]) if e is not None else p[pages, :, h:h + 1].double())
                    .reshape(-1, d)[:total] for p, e in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            for i in range(0, new, 1024):          # rows at a time: the scores in 64 bits take much room
                rows = slice(s["cuts"][b] + i, s["cuts"][b] + min(new, i + 1024))
                sc = s["q"][rows, heads].double().transpose(0, 1) @ k.t() / math.sqrt(d)
                sc.masked_fill_(hidden[i:i + 1024], float("-inf"))
                out[rows, heads] = (torch.softmax(sc, -1) @ v).transpose(0, 1)
    return out
