"""The 8-bit K/V cache and the attention over it, as they are measured.

Four operators (``csahca_amd.native``):

* ``write``   K and V of new tokens quantised into a paged cache, with one scale
              for each page and head (``kv8_write``);
* ``read``    tokens of that cache read back (``kv8_read``);
* ``attend``  attention over all of a sequence's cached tokens, one or several
              query tokens, grouped query heads (``kv8_decode_forward``);
* ``csa``     attention over the chunks that were selected
              (``kv8_csa_decode_forward``).

The cache: ``k_cache [pages, heads, page, D]``, ``v_cache [pages, heads,
page / 16, D, 16]`` (transposed in groups of 16 tokens), ``float8_e4m3fn`` or
``int8``, and fp32 scales ``[pages, heads]``, powers of two.  ``block_table[b,
j]`` is the page of sequence b's tokens ``[j * page, (j + 1) * page)``.

``own`` chooses between the library's kernels and the plain torch form.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
LEAST_EXP = -120  # exponent of the scale of an all-zero page
GROUP = 16  # tokens that v_cache holds together


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _write(name, B, N, held, *, Hkv=8, D=128, page=64, fmt="e4m3", dtype="bf16", ragged=False, packed=True):
    return dict(name=name, op="write", B=B, N=N, held=held, Hkv=Hkv, D=D, page=page, fmt=fmt, dtype=dtype,
                ragged=ragged, packed=packed)


def _read(name, B, S, *, Hkv=8, D=128, page=64, fmt="e4m3", dtype="bf16", ragged=False):
    return dict(name=name, op="read", B=B, S=S, Hkv=Hkv, D=D, page=page, fmt=fmt, dtype=dtype, ragged=ragged)


def _attend(name, B, S, *, Q=1, Hkv=8, G=1, D=128, page=64, fmt="e4m3", dtype="bf16", ragged=False):
    return dict(name=name, op="attend", B=B, S=S, Q=Q, Hkv=Hkv, G=G, D=D, page=page, fmt=fmt, dtype=dtype,
                ragged=ragged)


def _csa(name, B, S, top_k, *, Hkv=8, G=1, D=128, page=64, chunk=64, fmt="e4m3", dtype="bf16", ragged=False):
    return dict(name=name, op="csa", B=B, S=S, top_k=top_k, Hkv=Hkv, G=G, D=D, page=page, chunk=chunk, fmt=fmt,
                dtype=dtype, ragged=ragged)


def listed():
    return [
        # A decode step of 32 sequences: one token each appended to the page it falls in.
        _write("write_b32_n1", 32, 1, 700),
        # Prefill: 4 prompts of 8192 tokens into fresh pages, K and V as slices of a QKV projection.
        _write("write_b4_n8192", 4, 8192, 0),
        # A prompt chunk of ragged lengths behind a prefix that ends inside a page; 5 heads of 96, fp32 values, int8.
        _write("write_b3_n777_odd", 3, 777, 1001, Hkv=5, D=96, page=48, fmt="int8", dtype="f32", ragged=True,
               packed=False),
        # Reading 4 contexts of 8192 tokens back, to build chunk summaries or move them to a 16-bit cache.
        _read("read_b4_s8192", 4, 8192),
        # The same of ragged odd lengths, int8, 3 heads of 192, to fp32.
        _read("read_b5_s1999_odd", 5, 1999, Hkv=3, D=192, page=32, fmt="int8", dtype="f32", ragged=True),
        # One sequence at a short context: the smallest decode call, where latency and launches count.
        _attend("attend_b1_s8k", 1, 8192),
        # A serving batch of ragged contexts up to 32768 tokens, four query heads to a K/V head.
        _attend("attend_b16_s32k_gqa4", 16, 32768, G=4, ragged=True),
        # Three tokens verified at once, 15 query heads over 3 of 64, f16 over int8, small pages, one empty sequence.
        _attend("attend_b6_q3_odd_f16", 6, 5003, Q=3, Hkv=3, G=5, D=64, page=16, fmt="int8", dtype="f16", ragged=True),
        # A full serving batch at long context.
        _attend("attend_b32_s32k", 32, 32768),
        # A prompt chunk of 512 tokens over the 16384 tokens held with it, four query heads to a K/V head.
        _attend("attend_b2_q512_s16k_gqa4", 2, 16384, Q=512, G=4),
        # The reference's benchmark shape: one sequence, 32768 tokens, top-8 of 512 chunks.
        _csa("csa_b1_s32k_k8", 1, 32768, 8),
        # A full serving batch with a wide selection.
        _csa("csa_b32_s32k_k32", 32, 32768, 32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges: batches 1-32, lengths 1-32768, 1-512
    query tokens, every value type, cache format, head size and group of the
    operators, and no more work than the largest listed cases."""
    most = {c["op"]: 0 for c in listed()}
    for c in listed():
        most[c["op"]] = max(most[c["op"]], _cost(c))
    while True:
        case = _any(rng)
        if _cost(case) <= most[case["op"]] and _cached(case) <= 1 << 30 and _scores(case) <= 1 << 29:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 100)


def _cached(case):
    """Values of K that the plain form holds in fp32."""
    return 0 if case["op"] == "csa" else case["B"] * _blocks(case) * case["page"] * case["Hkv"] * case["D"]


def _scores(case):
    if case["op"] == "csa":
        return case["B"] * case["Hkv"] * case["top_k"] * case["chunk"] * (case["G"] + 2 * case["D"])
    return case["B"] * case["Hkv"] * case["G"] * case["Q"] * case["S"] if case["op"] == "attend" else 0


def _any(rng):
    op = rng.choice(["write", "write", "read", "attend", "attend", "attend", "csa", "csa"])
    case = dict(op=op, B=_log(rng, 1, 32), Hkv=rng.choice([1, 2, 3, 4, 5, 8, 8, 8]),
                D=rng.choice([64, 96, 128, 128, 128, 192, 256]), page=rng.choice([16, 32, 48, 64, 64, 64, 128, 256]),
                fmt=rng.choice(["e4m3", "e4m3", "int8"]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                ragged=rng.random() < 0.5)
    if op == "write":
        case.update(N=rng.choice([1, _log(rng, 1, 8192)]), held=rng.choice([0, _log(rng, 1, 4096)]),
                    packed=rng.random() < 0.5)
    elif op == "read":
        case.update(S=_log(rng, 1, 32768))
    elif op == "attend":
        case.update(S=_log(rng, 1, 32768), Q=rng.choice([1, 1, 1, _log(rng, 1, 512)]), G=rng.choice([1, 1, 2, 3, 4, 8]))
    else:
        chunk = rng.choice([16, 32, 48, 64, 64, 64, 100, 128])
        S = _log(rng, 256, 32768)
        case.update(S=S, G=rng.choice([1, 1, 2, 4]), chunk=chunk,
                    top_k=min(_log(rng, 1, 64), max(1, 4096 // chunk), max(1, S // chunk)))
    return case


def _counts(case):
    """Tokens of each sequence (new ones for a write): all alike, or ragged from
    a sixteenth of the largest up, the last one empty."""
    n, B = case["N"] if case["op"] == "write" else case["S"], case["B"]
    if not case["ragged"]:
        return [n] * B
    r = random.Random(n * 64 + B)
    lens = [n] + [min(n, _log(r, max(1, n // 16), n)) for _ in range(B - 1)]
    if B > 2:
        lens[-1] = 0
    return lens


def _held(case):
    """Tokens that each sequence of a write held before."""
    if not case["ragged"]:
        return [case["held"]] * case["B"]
    r = random.Random(case["held"])
    return [r.randint(0, case["held"]) for _ in range(case["B"])]


def _blocks(case):
    """Columns of the block table."""
    page = case["page"]
    if case["op"] == "write":  # the pages of the prefix and the new tokens, and one more
        return (case["held"] + case["N"] - 1) // page + 2
    return -(-case["S"] // page)


def _visible(case):
    """Query-key pairs of one query head, over the batch."""
    Q = case["Q"]
    return sum(max(0, n - Q + 1 + i) for n in _counts(case) for i in range(Q))


def work(case):
    B, H, D, page = case["B"], case["Hkv"], case["D"], case["page"]
    esz = DTYPES[case["dtype"]].itemsize
    lens = _counts(case)
    n = sum(lens)
    if case["op"] == "write":
        pages = sum((h + c - 1) // page - h // page + 1 for h, c in zip(_held(case), lens) if c)
        return {"bytes": 2 * n * H * D * (esz + 1) + 2 * 4 * pages * H + 8 * B, "flops": 6 * n * H * D}
    pages = sum(-(-x // page) for x in lens)
    if case["op"] == "read":
        out = 2 * B * case["S"] * H * D * esz  # the padding behind each sequence is written too
        return {"bytes": 2 * n * H * D + out + pages * (8 * H + 4), "flops": 2 * n * H * D}
    Q = case.get("Q", 1)
    io = 2 * B * Q * H * case["G"] * D * esz
    if case["op"] == "attend":
        return {"bytes": 2 * n * H * D + pages * (8 * H + 4) + io, "flops": 4 * D * H * case["G"] * _visible(case)}
    tokens = B * H * case["top_k"] * case["chunk"]
    return {"bytes": 2 * tokens * D + B * H * case["top_k"] * 16 + io, "flops": 4 * D * case["G"] * tokens}


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------
def _exponent(amax, fmt):
    """The least e with amax <= LARGEST 2^e, within the range of scales."""
    frac, exp = torch.frexp(amax)  # amax = frac 2^exp, frac in [0.5, 1)
    top, shift = math.frexp(LARGEST[fmt])
    e = torch.where(frac <= top, exp - shift, exp - shift + 1)
    return torch.where(amax > 0, e, torch.full_like(e, LEAST_EXP)).clamp(LEAST_EXP, -LEAST_EXP)


def _pow2(e):
    """2^e exactly, from the bits (a device's pow may be off in the last place)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to8(x, fmt):
    """fp32 values to 8 bits, to the nearest, ties to even."""
    x = x.clamp(-LARGEST[fmt], LARGEST[fmt])
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else x.round().to(torch.int8)


def _grouped(x):
    """[..., tokens, D] to v_cache's [..., tokens / 16, D, 16]."""
    return x.unflatten(-2, (-1, GROUP)).transpose(-1, -2)


def _ungrouped(x):
    return x.transpose(-1, -2).flatten(-3, -2)


def _values(shape, g, channels):
    """Keys or values as projections give them: normal, some channels larger."""
    return torch.randn(shape, device=DEV, generator=g) * channels


def _channels(D, g, wide):
    c = torch.ones(D, device=DEV)
    if wide:
        c[torch.randint(0, D, (max(1, D // 32),), device=DEV, generator=g)] = 4.0
    return c


def _cache(case, g):
    """A filled pool of pages, in an order of its own, and the block table."""
    B, H, D, page, fmt = case["B"], case["Hkv"], case["D"], case["page"], case["fmt"]
    M = _blocks(case)
    pages = B * M
    s = dict(table=torch.randperm(pages, device=DEV, generator=g).view(B, M).to(torch.int32))
    for name, shape, wide in (("k", (pages, H, page, D), True), ("v", (pages, H, page // GROUP, D, GROUP), False)):
        data = torch.empty(shape, dtype=FORMATS[fmt], device=DEV)
        scale = torch.empty(pages, H, device=DEV)
        ch = _channels(D, g, wide)
        step = max(1, (1 << 27) // (H * page * D))
        for p in range(0, pages, step):
            n = min(step, pages - p)
            x = _values((n, H, page, D), g, ch)
            e = _exponent(x.abs().amax((2, 3)), fmt)
            q = _to8(x * _pow2(-e)[..., None, None], fmt)
            q = q.view(torch.uint8)
            data.view(torch.uint8)[p : p + n] = q if name == "k" else _grouped(q)
            scale[p : p + n] = _pow2(e)
        s[name], s[name + "s"] = data, scale
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, H, D, dt = case["B"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    s = _cache(case, g)
    s["case"] = case
    lens = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
    if case["op"] == "write":
        N = case["N"]
        s["counts"] = lens if case["ragged"] else None
        s["start"] = torch.tensor(_held(case), dtype=torch.int32, device=DEV)
        x = torch.stack([_values((B, N, H, D), g, _channels(D, g, wide)).to(dt) for wide in (True, False)], 2)
        if case["packed"]:  # slices of one projection's [B, N, 2, H, D]
            s["knew"], s["vnew"] = x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2)
        else:
            s["knew"], s["vnew"] = (x[:, :, i].transpose(1, 2).contiguous() for i in (0, 1))
        return s
    s["lens"] = lens
    if case["op"] == "read":
        return s
    heads = H * case["G"]
    shape = (B, heads, D) if case["op"] == "csa" or case["Q"] == 1 else (B, case["Q"], heads, D)
    s["q"] = torch.randn(shape, device=DEV, generator=g).to(dt)
    if case["op"] == "csa":
        r = torch.rand(B, H, max(1, case["S"] // case["chunk"]), device=DEV, generator=g)
        s["ids"] = r.argsort(-1)[..., : case["top_k"]].to(torch.int32).contiguous()
    return s


# ---------------------------------------------------------------------------
# the calls
# ---------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


def _own_write(s):
    from csahca_amd import native

    native.kv8_write(s["knew"], s["vnew"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["start"], counts=s["counts"])
    return s["k"], s["v"], s["ks"], s["vs"]


def _own_read(s):
    from csahca_amd import native

    return native.kv8_read(s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"], s["case"]["S"],
                           dtype=DTYPES[s["case"]["dtype"]])


def _own_attend(s):
    from csahca_amd import native

    return native.kv8_decode_forward(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"])


def _own_csa(s):
    from csahca_amd import native

    return native.kv8_csa_decode_forward(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"], s["ids"],
                                         s["case"]["chunk"])


# The plain form.
def _plain_write(s):
    """The pages that the new tokens fall in, decoded, written and put back."""
    c = s["case"]
    B, N, page, fmt = c["B"], c["N"], c["page"], c["fmt"]
    dev = s["start"].device
    start = s["start"].long()
    count = torch.full((B,), N, device=dev) if s["counts"] is None else s["counts"].long()
    first = start // page
    pages = (N - 1) // page + 2  # as many as N tokens can touch, and the table has columns for
    pos = (first[:, None] * page + torch.arange(pages * page, device=dev)).view(B, pages, page)
    n = pos - start[:, None, None]
    new = (n >= 0) & (n < count[:, None, None])  # [B, pages, page]
    touched = new.any(-1)
    live = (n < 0) & touched[..., None]
    ids = s["table"].long().gather(1, first[:, None] + torch.arange(pages, device=dev))
    order = torch.arange(B, device=dev)[:, None, None]
    for x, data, scale in ((s["knew"], s["k"], s["ks"]), (s["vnew"], s["v"], s["vs"])):
        grouped = data.dim() == 5
        old8 = data.view(torch.uint8)[ids]
        old8 = (_ungrouped(old8) if grouped else old8).contiguous()  # [B, pages, H, page, D]
        old = old8.view(data.dtype).float()
        xn = x.transpose(1, 2)[order, n.clamp(0, N - 1)].float()  # [B, pages, page, H, D]
        xn = xn.transpose(2, 3)
        m = new[:, :, None, :, None]
        amax = torch.where(m, xn.abs(), 0.0).amax((3, 4))
        need = _pow2(_exponent(amax, fmt))
        s_old = scale[ids]
        has = live.any(-1)[..., None]
        s_new = torch.where(has, torch.maximum(s_old, need), need)
        s_new = torch.where(touched[..., None], s_new, s_old)
        again = _to8(old * (s_old / s_new)[..., None, None], fmt).view(torch.uint8)
        grown = live[:, :, None, :, None] & (s_new > s_old)[..., None, None]
        q = _to8(xn * (1.0 / s_new)[..., None, None], fmt).view(torch.uint8)
        q = torch.where(m, q, torch.where(grown, again, old8))
        q = _grouped(q) if grouped else q
        data.view(torch.uint8)[ids.flatten()] = q.flatten(0, 1)
        scale[ids.flatten()] = s_new.flatten(0, 1)
    return s["k"], s["v"], s["ks"], s["vs"]


def _plain_cached(s):
    """K and V of every sequence's table in fp32, [B, H, S, D]."""
    ids, S = s["table"].long(), s["case"]["S"]
    k = s["k"].view(torch.uint8)[ids].view(s["k"].dtype).float() * s["ks"][ids][..., None, None]
    k = k.transpose(1, 2).flatten(2, 3)[:, :, :S]
    v = s["v"].view(torch.uint8)[ids].view(s["v"].dtype).float() * s["vs"][ids][..., None, None, None]
    v = _ungrouped(v).transpose(1, 2).flatten(2, 3)[:, :, :S]
    return k, v


def _plain_read(s):
    k, v = _plain_cached(s)
    at = torch.arange(s["case"]["S"], device=k.device) < s["lens"][:, None]
    at = at[:, None, :, None]
    dt = DTYPES[s["case"]["dtype"]]
    return torch.where(at, k, 0.0).to(dt), torch.where(at, v, 0.0).to(dt)


def _softmax_times(score, see, v):
    """softmax over the seen, times v; 0 where nothing is seen."""
    score = torch.where(see, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(p, v) / total, 0.0)


def _plain_attend(s):
    c = s["case"]
    B, Q, H, G, D, S = c["B"], c["Q"], c["Hkv"], c["G"], c["D"], c["S"]
    k, v = _plain_cached(s)
    q = s["q"].float().view(B, Q, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, D)
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)
    last = s["lens"].long()[:, None] - Q + 1 + torch.arange(Q, device=q.device)  # tokens each query sees
    see = torch.arange(S, device=q.device) < last[..., None]  # [B, Q, S]
    see = see[:, None, :, None].expand(B, 1, Q, G, S).reshape(B, 1, Q * G, S)
    o = _softmax_times(score, see, v)
    return o.view(B, H, Q, G, D).permute(0, 2, 1, 3, 4).reshape(s["q"].shape).to(s["q"].dtype)


def _plain_csa(s):
    c = s["case"]
    B, H, G, D, page = c["B"], c["Hkv"], c["G"], c["D"], c["page"]
    tok = (s["ids"].long()[..., None] * c["chunk"] + torch.arange(c["chunk"], device=DEV)).flatten(2)  # [B, H, T]
    see = (tok >= 0) & (tok < s["lens"].long()[:, None, None])
    tok = tok.clamp(0, c["S"] - 1)
    ids = s["table"].long().gather(1, (tok // page).flatten(1)).view(tok.shape)
    off, h = tok % page, torch.arange(H, device=DEV)[None, :, None]
    k = s["k"].view(torch.uint8)[ids, h, off].view(s["k"].dtype).float() * s["ks"][ids, h][..., None]
    v = s["v"].view(torch.uint8)[ids, h, off // GROUP, :, off % GROUP].contiguous()
    v = v.view(s["v"].dtype).float() * s["vs"][ids, h][..., None]
    q = s["q"].float().view(B, H, G, D)
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)
    return _softmax_times(score, see[:, :, None], v).view(s["q"].shape).to(s["q"].dtype)


_PLAIN = {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "csa": _plain_csa}
_OWN = {"write": _own_write, "read": _own_read, "attend": _own_attend, "csa": _own_csa}


# ---------------------------------------------------------------------------
# the same in 64 bits, one sequence (and page or head) at a time
# ---------------------------------------------------------------------------
def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest(x, fmt):
    """fp64 values to the nearest that 8 bits hold, ties to even."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    step = _two_to((torch.frexp(x)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    if case["op"] == "write":
        # a page at a time: about 2 ms each
        return _exact_write(case, prepare(case, seed)) if sum(_counts(case)) < 4000 * case["page"] else None
    s = prepare(case, seed)
    lens, out = _counts(case), []
    for b in range(case["B"]):
        out.append(_EXACT[case["op"]](case, s, b, lens[b]))
    if case["op"] == "read":
        return torch.stack([o[0] for o in out]), torch.stack([o[1] for o in out])
    return torch.stack(out).view(s["q"].shape)


def _exact_write(case, s):
    page, fmt, D = case["page"], case["fmt"], case["D"]
    out = []
    for x, data, scale in ((s["knew"], s["k"], s["ks"]), (s["vnew"], s["v"], s["vs"])):
        val, sc, table = data.double(), scale.double(), s["table"].tolist()
        for b, (held, count) in enumerate(zip(_held(case), _counts(case))):
            n = 0
            while n < count:
                pos = held + n
                p, row = table[b][pos // page], pos % page
                m = min(page - row, count - n)
                new = x[b, :, n : n + m].double()  # [H, m, D]
                amax = new.abs().amax((1, 2))
                frac, e = torch.frexp(amax / LARGEST[fmt])
                e = torch.where(frac == 0.5, e - 1, e)
                # a quotient that rounded to a power of two from above
                e = torch.where(amax > LARGEST[fmt] * _two_to(e), e + 1, e)
                new_s = _two_to(torch.where(amax > 0, e, LEAST_EXP).clamp(LEAST_EXP, -LEAST_EXP))
                if row:
                    new_s = torch.maximum(new_s, sc[p])
                rows = val[p] if data.dim() == 4 else val[p].permute(0, 1, 3, 2).reshape(-1, page, D)
                rows = rows.clone()
                if row:
                    moved = _nearest(rows[:, :row] * (sc[p] / new_s)[:, None, None], fmt)
                    rows[:, :row] = torch.where((new_s > sc[p])[:, None, None], moved, rows[:, :row])
                rows[:, row : row + m] = _nearest(new / new_s[:, None, None], fmt)
                val[p] = rows if data.dim() == 4 else rows.view(-1, page // GROUP, GROUP, D).permute(0, 1, 3, 2)
                sc[p] = new_s
                n += m
        out.append((val, sc))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_tokens(case, s, b, n):
    """K and V of sequence b's first n tokens in fp64, [H, n, D]."""
    ids = s["table"][b, : -(-n // case["page"])].long()
    k = s["k"].view(torch.uint8)[ids].view(s["k"].dtype).double() * s["ks"].double()[ids][:, :, None, None]
    v = s["v"].view(torch.uint8)[ids].view(s["v"].dtype).double() * s["vs"].double()[ids][:, :, None, None, None]
    v = v.permute(1, 0, 2, 4, 3).reshape(case["Hkv"], -1, case["D"])
    return k.transpose(0, 1).reshape(case["Hkv"], -1, case["D"])[:, :n], v[:, :n]


def _exact_read(case, s, b, n):
    pad = torch.zeros(2, case["Hkv"], case["S"], case["D"], dtype=torch.float64, device=DEV)
    if n:
        pad[0, :, :n], pad[1, :, :n] = _exact_tokens(case, s, b, n)
    return pad


def _exact_attend(case, s, b, n):
    Q, H, G, D = case["Q"], case["Hkv"], case["G"], case["D"]
    q = s["q"][b].double().view(Q, H, G, D)
    o = torch.zeros_like(q)
    if n:
        k, v = _exact_tokens(case, s, b, n)
        for h in range(H):
            score = q[:, h].reshape(Q * G, D) @ k[h].T / math.sqrt(D)
            gone = torch.arange(n, device=DEV) >= n - Q + 1 + torch.arange(Q, device=DEV).repeat_interleave(G)[:, None]
            p = torch.softmax(score.masked_fill(gone, -math.inf), -1)
            o[:, h] = torch.nan_to_num(p @ v[h]).view(Q, G, D)  # a query that sees nothing: 0
    return o


def _exact_csa(case, s, b, n):
    H, G, D, chunk = case["Hkv"], case["G"], case["D"], case["chunk"]
    q = s["q"][b].double().view(H, G, D)
    o = torch.zeros_like(q)
    if n:
        k, v = _exact_tokens(case, s, b, n)
        for h in range(H):
            tok = (s["ids"][b, h].long()[:, None] * chunk + torch.arange(chunk, device=DEV)).flatten()
            tok = tok[tok < n]
            if tok.numel():
                p = torch.softmax(q[h] @ k[h, tok].T / math.sqrt(D), -1)
                o[h] = p @ v[h, tok]
    return o


_EXACT = {"read": _exact_read, "attend": _exact_attend, "csa": _exact_csa}
