"""Serving operators for long contexts and 8-bit projections, as cases to be timed and compared.

Five operators of one decode step of a server whose cache is held in 4 bits: a projection in 8-bit
integers with a scale for each token and channel ("product"), rotary positions of its rows ("rope"),
new rows quantised into 4-bit pages and read back ("append"), one new token per sequence attending
over its pages and leaving its weight on them ("attention"), and the rows of least accumulated weight
left behind when a sequence outgrows its budget ("evict").

With ``own`` false ``run`` computes them from elementary torch operations; with ``own`` true it calls
the entry points of libjieyu_b200.so.
"""
import math

import numpy as np
import torch

own = False

# ---------------------------------------------------------------------------------------------------
# Cases


def listed():
    return [
        # one decode step of 64 sequences: query and key heads of fused rows, halves layout
        dict(name="rope_64x40x128", op="rope", rows=64, heads=40, hd=128, rot=128, halves=True, context=4352,
             padding=0),
        # a prompt of 16384 rows, interleaved pairs over half of each head, padding rows among them
        dict(name="rope_16384x40x128_part", op="rope", rows=16384, heads=40, hd=128, rot=64, halves=False,
             context=131072, padding=111),
        # the next token of eight sequences goes into their pages: pure latency
        dict(name="append_8x8x128", op="append", rows=8, seqs=8, kv=8, hd=128, page=16, context=2304, rot=128,
             halves=True, heads_first=False, padding=0),
        # the prompts of four sequences written in one call, padding rows among them
        dict(name="append_16384x8x128", op="append", rows=16384, seqs=4, kv=8, hd=128, page=64, context=4352, rot=128,
             halves=False, heads_first=False, padding=37),
        # the smallest step: one short sequence, 14 query heads on 2 kv heads of 64
        dict(name="attention_1x513_14x2x64", op="attention", seqs=1, longest=513, shortest=513, empty=0, heads=14,
             kv=2, hd=64, page=16, rot=64, halves=True, heads_first=False, mass=False),
        # ragged lengths from one token to 8192 and empty places of the batch; weights are gathered
        dict(name="attention_48xragged_32x8x128", op="attention", seqs=48, longest=8192, shortest=1, empty=3,
             heads=32, kv=8, hd=128, page=64, rot=0, halves=False, heads_first=True, mass=True),
        # one very long sequence: all the parallelism has to come from the cache's length
        dict(name="attention_1x131072_32x8x128", op="attention", seqs=1, longest=131072, shortest=131072, empty=0,
             heads=32, kv=8, hd=128, page=64, rot=128, halves=False, heads_first=False, mass=False),
        # a batch a little over its budget, as a server trims it every few hundred steps
        dict(name="evict_16x2304_to_2048", op="evict", seqs=16, longest=2304, shortest=1900, empty=0, budget=2048,
             recent=256, kv=8, hd=64, page=32, heads_first=False),
        # one long context cut to an eighth
        dict(name="evict_1x131072_to_16384", op="evict", seqs=1, longest=131072, shortest=131072, empty=0,
             budget=16384, recent=1024, kv=8, hd=128, page=64, heads_first=False),
        # one token through a square projection: the weights are all there is to read
        dict(name="product_1x4096x4096", op="product", m=1, n=4096, k=4096, bias=False),
        # a batch of 48 tokens through a wide projection with an odd depth
        dict(name="product_48x14336x4090", op="product", m=48, n=14336, k=4090, bias=True),
        # a prompt of 4096 tokens through the feed-forward's projection
        dict(name="product_4096x14336x4096", op="product", m=4096, n=14336, k=4096, bias=False),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def _head(rng):
    return rng.choice([4 * rng.randint(2, 64), 64, 80, 96, 128, 256])


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention", "evict", "product", "product"])
    if op == "product":
        n, k = _log(rng, 16, 16384), _log(rng, 16, 16384)
        most = max(1, min(4096, 4096 * 14336 * 4096 // (n * k)))
        return dict(op=op, m=_log(rng, 1, most), n=n, k=k, bias=rng.random() < 0.5)
    hd = _head(rng)
    rot = rng.choice([hd, hd, hd // 2 // 2 * 2, 2 * rng.randint(1, hd // 2)])
    halves = rng.random() < 0.5
    if op == "rope":
        heads = rng.randint(1, 48)
        return dict(op=op, rows=_log(rng, 1, max(1, min(16384, 16384 * 40 * 128 // (heads * hd)))), heads=heads,
                    hd=hd, rot=rot, halves=halves, context=_log(rng, 16, 131072), padding=rng.choice([0, 0, 1]))
    kv = rng.randint(1, 16)
    page, heads_first = rng.choice([1, 7, 16, 32, 64, 128, 257]), rng.random() < 0.5
    if op == "append":
        rows = min(_log(rng, 1, 16384), 16384 * 8 * 128 // (kv * hd))
        seqs = rng.randint(1, min(rows, 64))
        return dict(op=op, rows=rows, seqs=seqs, kv=kv, hd=hd, page=page, context=-(-rows // seqs) + rng.randint(0, 300),
                    rot=rng.choice([0, rot]), halves=halves, heads_first=heads_first,
                    padding=rng.choice([0, 0, rng.randint(0, rows // 4)]))
    if op == "evict":
        seqs = _log(rng, 1, 64)
        longest = _log(rng, 4, max(8, min(131072, 131072 * 8 * 128 // (seqs * kv * hd))))
        budget = rng.randint(1, max(1, min(longest, 16384 * 8 * 128 // (seqs * kv * hd))))
        return dict(op=op, seqs=seqs, longest=longest, shortest=rng.randint(1, longest),
                    empty=rng.choice([0, 0, rng.randint(0, seqs - 1)]), budget=budget, recent=rng.randint(0, budget),
                    kv=kv, hd=hd, page=page, heads_first=heads_first)
    kv, group = rng.randint(1, 8), rng.choice([1, 2, 4, 7, 8, 12, 16, 24])
    seqs = _log(rng, 1, 128)
    most = max(8, 131072 * 8 * 128 // (seqs * kv * hd))
    longest = _log(rng, 1, min(most, 131072, max(1, 40_000_000 // (seqs * kv * group))))
    return dict(op=op, seqs=seqs, longest=longest, shortest=rng.randint(1, longest),
                empty=rng.choice([0, 0, rng.randint(0, seqs - 1)]), heads=kv * group, kv=kv, hd=hd, page=page,
                rot=rng.choice([0, rot]), halves=halves, heads_first=heads_first, mass=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------
# Inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tables(positions, rot):
    """cos and sin [positions][rot / 2], theta 5e5 (angles in 64 bits)."""
    j = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * 5e5 ** (-2.0 * j / rot)
    return angle.cos().float(), angle.sin().float()


def _groups(hd):
    return -(-hd // 32)


def _new_pool(case, gen, pages):
    kv, page, groups = case["kv"], case["page"], _groups(case["hd"])
    shape = (pages, kv, page) if case["heads_first"] else (pages, page, kv)
    return {"num_pages": pages, "page": page, "heads_first": case["heads_first"],
            "k": torch.zeros(shape + (16 * groups,), dtype=torch.uint8, device="cuda"),
            "v": torch.zeros(shape + (16 * groups,), dtype=torch.uint8, device="cuda"),
            "kp": torch.zeros(shape + (groups, 2), dtype=torch.float16, device="cuda"),
            "vp": torch.zeros(shape + (groups, 2), dtype=torch.float16, device="cuda"),
            "mass": torch.zeros(shape, device="cuda")}


def _fill(pool, hd, gen):
    """What quantised rows look like: steps of a 4-bit grid, the lowest value about eight steps below zero."""
    left = hd % 32
    for name in ("k", "v"):
        for a in pool[name].split(max(1, (1 << 26) // pool[name][0].numel())):
            a.copy_(torch.randint(0, 256, a.shape, generator=gen, device="cuda", dtype=torch.uint8))
        if left:  # dims behind the head's last one are stored as zero
            last = pool[name][..., -16:]
            at = torch.arange(16, device="cuda")
            mask = (at < left).to(torch.uint8) * 15 + (at + 16 < left).to(torch.uint8) * 240
            last.bitwise_and_(mask)
        p = pool[name + "p"]
        step = 0.05 + 0.3 * torch.rand(p.shape[:-1], generator=gen, device="cuda")
        p[..., 0] = step
        p[..., 1] = -step * (6.5 + 2 * torch.rand(p.shape[:-1], generator=gen, device="cuda"))


def _table(gen, pages, seqs, width):
    order = torch.randperm(pages, generator=gen, device="cuda")[: seqs * width]
    return order.to(torch.int32).reshape(seqs, width).contiguous()


def _lengths(case, gen):
    lens = torch.randint(case["shortest"], case["longest"] + 1, (case["seqs"],), generator=gen, device="cuda")
    lens[torch.randint(0, case["seqs"], (1,), generator=gen, device="cuda")] = case["longest"]
    if case["empty"]:
        lens[torch.randperm(case["seqs"], generator=gen, device="cuda")[: case["empty"]]] = 0
    return lens.to(torch.int32)


def _prepare_pages(case, state, gen):
    op, kv, hd, seqs = case["op"], case["kv"], case["hd"], case["seqs"]
    width = -(-(case["context"] if op == "append" else case["longest"]) // case["page"])
    new_width = -(-case["budget"] // case["page"]) if op == "evict" else 0
    need = seqs * (width + new_width)
    pool = state["pool"] = _new_pool(case, gen, need + need // 4 + 1)
    tables = _table(gen, pool["num_pages"], seqs, width + new_width)
    pool["table"], pool["width"] = tables[:, :width].contiguous(), width
    if op != "append":
        _fill(pool, hd, gen)
        state["lens"] = _lengths(case, gen)
    if op == "evict":
        state["new_table"] = tables[:, width:].contiguous()
        state["new_lens"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        state["kept"] = torch.zeros(seqs, kv, case["budget"], dtype=torch.int32, device="cuda")
        # accumulated weights: a few heavy rows, most light, many equal
        mass = (2.5 * torch.randn(pool["mass"].shape, generator=gen, device="cuda")).exp()
        mass[torch.rand(mass.shape, generator=gen, device="cuda") < 0.3] = 0.0
        pool["mass"].copy_(mass)
        rows = seqs * case["budget"]
        state["back_seq"] = torch.arange(seqs, device="cuda").repeat_interleave(case["budget"]).to(torch.int32)
        at = torch.arange(case["budget"], device="cuda").repeat(seqs)
        there = torch.minimum(state["lens"], torch.tensor(case["budget"], device="cuda"))
        at[at >= there[state["back_seq"].long()]] = -1
        state["back_pos"] = at.to(torch.int32)
    if op == "append":
        rows = case["rows"]
        i = torch.arange(rows, device="cuda")
        room = case["context"] - -(-rows // seqs)
        start = torch.randint(0, room + 1, (seqs,), generator=gen, device="cuda")
        seq, order = (i % seqs).sort(stable=True)
        pos = start[seq] + (i // seqs)[order]
        if case["padding"]:
            pos[torch.randperm(rows, generator=gen, device="cuda")[: case["padding"]]] = -1
        state["seq"], state["pos"] = seq.to(torch.int32), pos.to(torch.int32)
        # the key and value columns of a fused projection's rows
        fused = torch.randn(rows, 2 * kv * hd, generator=gen, device="cuda")
        state["k"], state["v"] = fused[:, : kv * hd], fused[:, kv * hd:]
    if op in ("append", "evict"):
        state["k_back"] = torch.zeros(rows, kv * hd, device="cuda")
        state["v_back"] = torch.zeros(rows, kv * hd, device="cuda")
    if op == "attention":
        state["q"] = 2.0 * torch.randn(seqs, case["heads"] * hd, generator=gen, device="cuda")
        state["out"] = torch.zeros_like(state["q"])
        # the new token's position: rows that were evicted before leave it behind the length
        state["turn"] = (state["lens"] - 1 + 5).clamp(min=0).to(torch.int32)
    if case.get("rot"):
        state["cos"], state["sin"] = _tables((case["context"] if op == "append" else case["longest"]) + 8, case["rot"])


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": case}
    op = case["op"]
    if op == "rope":
        rows, width = case["rows"], case["heads"] * case["hd"]
        state["x"] = torch.randn(rows, width, generator=gen, device="cuda")
        state["y"] = torch.zeros(rows, width, device="cuda")
        pos = torch.randint(0, case["context"], (rows,), generator=gen, device="cuda")
        if case["padding"]:
            pos[torch.randperm(rows, generator=gen, device="cuda")[: case["padding"]]] = -1
        state["pos"] = pos.to(torch.int32)
        state["cos"], state["sin"] = _tables(case["context"], case["rot"])
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        pitch = -(-k // 16) * 16
        x = torch.randn(m, k, generator=gen, device="cuda")
        hot = torch.randint(0, k, (max(1, k // 500),), generator=gen, device="cuda")
        x[:, hot] *= 12  # a few channels of activations stand out
        state["x"] = x
        state["w"] = torch.zeros(n, pitch, dtype=torch.int8, device="cuda")
        state["w"][:, :k] = (40 * torch.randn(n, k, generator=gen, device="cuda")).round().clamp(-127, 127)
        state["ws"] = 2e-4 + 4e-4 * torch.rand(n, generator=gen, device="cuda")
        if case["bias"]:
            state["bias"] = torch.randn(n, generator=gen, device="cuda")
        state["a"] = torch.zeros(m, pitch, dtype=torch.int8, device="cuda")
        state["as"] = torch.zeros(m, device="cuda")
        state["y"] = torch.zeros(m, n, device="cuda")
    else:
        _prepare_pages(case, state, gen)
    return state


# ---------------------------------------------------------------------------------------------------
# The plain forms


def _turn(x, pos, cos, sin, halves):
    """x [rows, heads, hd], its first 2 * cos.shape[1] dims rotated by the row's position: two products, the second
    rounded, one fused sum."""
    half = cos.shape[1]
    c, s = cos[pos][:, None].double(), sin[pos][:, None].double()
    part = x[..., : 2 * half].double()
    a, b = (part[..., :half], part[..., half:]) if halves else (part[..., 0::2], part[..., 1::2])
    r0 = (a * c - (b * s).float().double()).float()
    r1 = (a * s + (b * c).float().double()).float()
    turned = torch.cat((r0, r1), -1) if halves else torch.stack((r0, r1), -1).flatten(-2)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _eight(x):
    """Whole numbers in -127..127 (as floats) and one scale for each last axis."""
    amax = x.abs().amax(-1, keepdim=True)
    c127 = torch.full_like(amax, 127.0)
    zero = torch.zeros_like(amax)
    inverse = torch.where(amax > 1e-8, c127 / amax, zero)
    scale = torch.where(amax > 1e-8, amax / c127, zero)
    return (x * inverse).clamp(-127.0, 127.0).round(), scale


def _four(x):
    """4-bit numbers [.., groups, 32] with their groups' step and lowest value (fp16, as floats) of x [.., hd]."""
    hd, groups = x.shape[-1], _groups(x.shape[-1])
    pad = 32 * groups - hd
    spread = lambda fill: torch.nn.functional.pad(x, (0, pad), value=fill).unflatten(-1, (groups, 32))  # noqa: E731
    low, high = (a.clamp(-65504.0, 65504.0) for a in (spread(math.inf).amin(-1), spread(-math.inf).amax(-1)))
    step = ((high - low) / torch.full_like(low, 15.0)).half().float()
    low = low.half().float()
    inverse = torch.where(step > 0, 1.0 / step, 0.0)
    q = ((spread(0.0) - low[..., None]) * inverse[..., None]).round().clamp(0, 15)
    if pad:
        q.flatten(-2)[..., hd:] = 0
    return q, step, low


def _places(pool, names):
    """The pool's arrays as [pages, positions, kv heads, ...] whatever their order in memory."""
    return [pool[n].transpose(1, 2) if pool["heads_first"] else pool[n] for n in names]


def _values(bytes_, params, hd):
    """fp32 values of stored rows [.., 16 groups] with params [.., groups, 2]."""
    b = bytes_.unflatten(-1, (-1, 16))
    q = torch.cat((b & 15, b >> 4), -1).float()
    p = params.float()
    return (p[..., :1] * q + p[..., 1:]).flatten(-2)[..., :hd]


def _find(pool, table, seq, pos):
    return table[seq, pos // pool["page"]].long(), pos % pool["page"]


def _plain_read(state, table, seq, pos):
    case, pool = state["case"], state["pool"]
    live = pos >= 0
    page, slot = _find(pool, table, seq[live].long(), pos[live].long())
    for name in ("k", "v"):
        x, p = _places(pool, (name, name + "p"))
        state[name + "_back"][live] = _values(x[page, slot], p[page, slot], case["hd"]).flatten(1)


def _plain_append(state):
    case, pool = state["case"], state["pool"]
    live = state["pos"] >= 0
    pos = state["pos"][live].long()
    page, slot = _find(pool, pool["table"], state["seq"][live].long(), pos)
    k, v = (state[n][live].reshape(-1, case["kv"], case["hd"]) for n in ("k", "v"))
    if "cos" in state:
        k = _turn(k, pos, state["cos"], state["sin"], case["halves"])
    for name, x in (("k", k), ("v", v)):
        to, params = _places(pool, (name, name + "p"))
        q, step, low = _four(x)
        to[page, slot] = (q[..., :16] + 16 * q[..., 16:]).flatten(-2).to(torch.uint8)
        params[page, slot] = torch.stack((step, low), -1).half()
    _places(pool, ("mass",))[0][page, slot] = 0.0


def _plain_attention(state):
    case, pool, lens = state["case"], state["pool"], state["lens"].long()
    seqs, heads, kv, hd = case["seqs"], case["heads"], case["kv"], case["hd"]
    q = state["q"].reshape(seqs, heads, hd)
    if "cos" in state:
        q = _turn(q, state["turn"].long(), state["cos"], state["sin"], case["halves"])
    q, qs = _eight(q)
    at = torch.arange(case["longest"], device="cuda")
    page, slot = pool["table"][:, at // pool["page"]].long(), at % pool["page"]
    pk, pkp, pv, pvp, pm = _places(pool, ("k", "kp", "v", "vp", "mass"))
    k = _values(pk[page, slot], pkp[page, slot], hd).permute(0, 2, 1, 3)  # [seqs, kv, positions, hd]
    q, qs = q.reshape(seqs, kv, -1, hd), qs.reshape(seqs, kv, -1, 1)
    scores = (q @ k.transpose(-1, -2)) * (qs * (1.0 / math.sqrt(hd)))
    here = (at < lens[:, None])[:, None, None]
    scores = torch.where(here, scores, -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(m == -math.inf, 0.0, m)).exp()
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = _values(pv[page, slot], pvp[page, slot], hd).permute(0, 2, 1, 3)
    state["out"].copy_((p @ v).reshape(seqs, -1))
    if case["mass"]:
        live = (at < lens[:, None]).nonzero(as_tuple=True)
        pm[page[live], slot.expand(seqs, -1)[live]] += p.sum(2).transpose(1, 2)[live]


def _plain_evict(state):
    case, pool, lens = state["case"], state["pool"], state["lens"].long()
    budget = case["budget"]
    at = torch.arange(case["longest"], device="cuda")
    page, slot = pool["table"][:, at // pool["page"]].long(), at % pool["page"]
    mass = _places(pool, ("mass",))[0][page, slot].transpose(1, 2)  # [seqs, kv, positions]
    n = lens[:, None, None]
    mass = torch.where(at < n, torch.where(at >= n - case["recent"], math.inf, mass), -math.inf)
    order = mass.argsort(dim=-1, descending=True, stable=True)[..., :budget]
    there = torch.arange(order.shape[-1], device="cuda") < n
    order = torch.where(there, order, case["longest"]).sort(-1).values
    kept = torch.full_like(state["kept"], -1)
    kept[..., : order.shape[-1]] = torch.where(order < case["longest"], order, -1)
    state["kept"].copy_(kept)
    state["new_lens"].copy_(lens.clamp(max=budget))
    seq, head, to = (kept >= 0).nonzero(as_tuple=True)
    source = kept[seq, head, to].long()
    sp, ss = _find(pool, pool["table"], seq, source)
    dp, ds = _find(pool, state["new_table"], seq, to)
    for x in _places(pool, ("k", "kp", "v", "vp", "mass")):
        x[dp, ds, head] = x[sp, ss, head]


def _plain_product(state):
    case = state["case"]
    q, scale = _eight(state["x"])
    y = torch.zeros(case["m"], case["n"], dtype=torch.int32, device="cuda")
    for i in range(0, case["k"], 1024):  # sums of 1024 products of 7 bits are whole in 32-bit floats
        j = min(case["k"], i + 1024)
        y += (q[:, i:j] @ state["w"][:, i:j].float().T).to(torch.int32)
    y = y.float() * (scale * state["ws"])
    state["y"].copy_(y + state["bias"] if case["bias"] else y)


def _plain_rope(state):
    case = state["case"]
    live = state["pos"] >= 0
    x = state["x"][live].reshape(-1, case["heads"], case["hd"])
    state["y"][live] = _turn(x, state["pos"][live].long(), state["cos"], state["sin"], case["halves"]).flatten(1)


# ---------------------------------------------------------------------------------------------------
# The framework's calls


def _kv_pages(pool, with_mass):
    from jieyu_b200 import _capi
    k, p, m = pool["k"], pool["kp"], pool["mass"]
    a, b = (2, 1) if pool["heads_first"] else (1, 2)
    return _capi.KVPagesQ4(k.data_ptr(), p.data_ptr(), pool["v"].data_ptr(), pool["vp"].data_ptr(),
                           m.data_ptr() if with_mass else None, pool["num_pages"], pool["page"],
                           k.stride(0), k.stride(a), k.stride(b), p.stride(0) // 2, p.stride(a) // 2, p.stride(b) // 2,
                           m.stride(0), m.stride(a), m.stride(b))


def _at(state, name):
    return state[name].data_ptr() if name in state else None


def _calls(state):
    """The calls of one pass as (function, arguments before the stream): a program makes them once per buffer set."""
    import ctypes

    from jieyu_b200 import _capi
    lib, case = _capi.load(), state["case"]
    op = case["op"]
    rope = None
    if "cos" in state:
        state["rope"] = _capi.Rope(_at(state, "cos"), _at(state, "sin"), state["cos"].shape[0], case["rot"],
                                   _capi.JYC_ROPE_HALVES if case["halves"] else _capi.JYC_ROPE_PAIRS)
        rope = ctypes.byref(state["rope"])
    if op == "rope":
        return [(lib.jyc_rope_rows, (_at(state, "x"), state["x"].stride(0), _at(state, "y"), state["y"].stride(0),
                                     case["rows"], case["heads"], case["hd"], _at(state, "pos"), rope))]
    if op == "product":
        a, w, m, n, k = state["a"], state["w"], case["m"], case["n"], case["k"]
        return [(lib.jyc_quantize_rows_i8, (_at(state, "x"), state["x"].stride(0), m, k, _at(state, "a"), a.stride(0),
                                            _at(state, "as"))),
                (lib.jyc_matmul_i8, (_at(state, "a"), a.stride(0), _at(state, "as"), _at(state, "w"), w.stride(0),
                                     _at(state, "ws"), _at(state, "bias"), _at(state, "y"), state["y"].stride(0),
                                     m, n, k))]
    pool, kv, hd = state["pool"], case["kv"], case["hd"]
    state["pages"] = _kv_pages(pool, op != "attention" or case["mass"])
    pages = ctypes.byref(state["pages"])
    table = (pool["table"].data_ptr(), pool["width"], case["seqs"])
    if op == "attention":
        need = lib.jyc_attention_paged_q4_workspace(case["seqs"], case["heads"], kv, hd,
                                                    pool["width"] * pool["page"] if case["mass"] else 0)
        state["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        return [(lib.jyc_attention_paged_q4,
                 (_at(state, "q"), state["q"].stride(0), _at(state, "out"), state["out"].stride(0), case["heads"],
                  kv, hd, _at(state, "lens")) + table
                 + (rope, _at(state, "turn"), pages, state["workspace"].data_ptr(), need))]
    back = (_at(state, "k_back"), _at(state, "v_back"), state["k_back"].stride(0))
    if op == "evict":
        new = (_at(state, "new_table"), state["new_table"].shape[1])
        rows = (state["back_pos"].numel(), kv, hd, _at(state, "back_seq"), _at(state, "back_pos"))
        return [(lib.jyc_kv_evict_paged_q4,
                 (_at(state, "lens"), case["budget"], case["recent"], kv, hd) + table
                 + new + (_at(state, "new_lens"), _at(state, "kept"), pages)),
                (lib.jyc_kv_read_paged_q4, back + rows + new + (case["seqs"], pages))]
    rows = (case["rows"], kv, hd, _at(state, "seq"), _at(state, "pos"))
    return [(lib.jyc_kv_append_paged_q4, (_at(state, "k"), _at(state, "v"), state["k"].stride(0)) + rows + table
             + (rope, None, pages)),
            (lib.jyc_kv_read_paged_q4, back + rows + table + (pages,))]


def run(state):
    """One pass. What an append or an eviction writes is held in 4 bits: the rows come back as the values they
    stand for, through the read operator, which is part of the pass. Weights are gathered from none, as in the
    first step after a reset."""
    case = state["case"]
    op = case["op"]
    if op == "attention" and case["mass"]:
        state["pool"]["mass"].zero_()
    if own:
        if "calls" not in state:
            state["calls"] = _calls(state)
        stream = torch.cuda.current_stream().cuda_stream
        for call, arguments in state["calls"]:
            status = call(*arguments, stream)
            if status < 0:
                raise RuntimeError("status %d" % status)
    elif op == "rope":
        _plain_rope(state)
    elif op == "product":
        _plain_product(state)
    elif op == "attention":
        _plain_attention(state)
    elif op == "append":
        _plain_append(state)
        _plain_read(state, state["pool"]["table"], state["seq"], state["pos"])
    else:
        _plain_evict(state)
        _plain_read(state, state["new_table"], state["back_seq"], state["back_pos"])
    if op in ("rope", "product"):
        return {"y": state["y"]}
    if op == "attention":
        out = {"out": state["out"]}
        if case["mass"]:
            out["mass"] = state["pool"]["mass"]
        return out
    out = {"k": state["k_back"], "v": state["v_back"]}
    if op == "evict":
        out["kept"], out["lens"] = state["kept"], state["new_lens"]
    return out


# ---------------------------------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 4 * m * k + n * k + 4 * n + 4 * m * n, "flops": 2 * m * n * k}
    hd = case["hd"]
    if op == "rope":
        rows = max(1, case["rows"] - case["padding"])
        tables = 4 * case["rot"] * min(rows, case["context"])
        return {"bytes": 8 * rows * case["heads"] * hd + tables, "flops": 3 * rows * case["heads"] * case["rot"]}
    kv = case["kv"]
    stored, floats = 40 * _groups(hd) * kv, 8 * hd * kv  # bytes of a row's K and V in the cache, and as fp32
    if op == "append":
        rows = max(1, case["rows"] - case["padding"])
        tables = 4 * case["rot"] * min(rows, case["context"])
        return {"bytes": 2 * rows * (stored + floats) + 4 * rows * kv + tables + 16 * case["rows"],
                "flops": 16 * rows * kv * hd}
    live = case["seqs"] - case["empty"]
    tokens = live * (case["longest"] + case["shortest"]) / 2
    if op == "attention":
        mass = 4 * tokens * kv if case["mass"] else 0
        return {"bytes": tokens * stored + mass + 4 * tokens / case["page"] + 8 * case["seqs"] * case["heads"] * hd,
                "flops": 4 * tokens * case["heads"] * hd}
    rows = live * min(case["budget"], (case["longest"] + case["shortest"]) / 2)
    return {"bytes": 4 * tokens * kv + rows * (3 * stored + floats + 12 * kv), "flops": tokens * kv + 4 * rows * kv * hd}


# ---------------------------------------------------------------------------------------------------
# The definitions in 64 bits. The whole numbers of 8 and 4 bits, their scales, steps and lowest values are
# roundings by definition (to fp32, or to fp16 from fp32), made here by rounding 64-bit results.


def _f32(x):
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def _f16(x):
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float16).astype(np.float64)


def _np(x):
    x = x.cpu().numpy()
    return x.astype(np.float64) if x.dtype.kind == "f" else x.astype(np.int64)


def _turned(x, pos, cos, sin, halves, rounded):
    """Rotation pair by pair; rounded where its result is quantised next."""
    near = _f32 if rounded else (lambda a: a)
    out = x.copy()
    half = cos.shape[1]
    for p in range(half):
        i, j = (p, p + half) if halves else (2 * p, 2 * p + 1)
        c, s = cos[pos, p][:, None], sin[pos, p][:, None]
        out[:, :, i] = near(x[:, :, i] * c - near(x[:, :, j] * s))
        out[:, :, j] = near(x[:, :, i] * s + near(x[:, :, j] * c))
    return out


def _int8(x):
    amax = np.max(np.abs(x), axis=-1, keepdims=True)
    tiny = amax <= np.float64(np.float32(1e-8))
    safe = np.where(tiny, 1.0, amax)
    inverse, scale = np.where(tiny, 0.0, _f32(127.0 / safe)), np.where(tiny, 0.0, _f32(safe / 127.0))
    return np.rint(np.clip(_f32(x * inverse), -127, 127)), scale


def _through_four_bits(x):
    """The values that x [rows, heads, hd] stands for once it is stored."""
    out = np.empty_like(x)
    for d in range(0, x.shape[-1], 32):
        g = x[..., d: d + 32]
        low, high = (np.clip(a, -65504.0, 65504.0) for a in (g.min(-1, keepdims=True), g.max(-1, keepdims=True)))
        step, base = _f16(_f32(_f32(high - low) / 15.0)), _f16(low)
        inverse = np.where(step > 0, _f32(1.0 / np.where(step > 0, step, 1.0)), 0.0)
        q = np.clip(np.rint(_f32(_f32(g - base) * inverse)), 0, 15)
        out[..., d: d + 32] = base + step * q
    return out


def _stored(bytes_, params, hd):
    """Torch, 64 bits: the values of stored rows."""
    out = torch.empty(bytes_.shape[:-1] + (hd,), dtype=torch.float64, device=bytes_.device)
    for d in range(hd):
        group, i = divmod(d, 32)
        byte = bytes_[..., 16 * group + i % 16].long()
        nibble = byte % 16 if i < 16 else torch.div(byte, 16, rounding_mode="floor")
        out[..., d] = params[..., group, 0].double() * nibble + params[..., group, 1].double()
    return out


def _exact_append(state, case):
    pos = _np(state["pos"])
    live = pos >= 0
    found = {}
    for name in ("k", "v"):
        x = _np(state[name]).reshape(case["rows"], case["kv"], case["hd"])[live]
        if name == "k" and "cos" in state:
            x = _turned(x, pos[live], _np(state["cos"]), _np(state["sin"]), case["halves"], True)
        back = np.zeros((case["rows"], case["kv"] * case["hd"]))
        back[live] = _through_four_bits(x).reshape(len(x), -1)
        found[name] = back
    return found


def _exact_attention(state, case):
    lens, pool, page = _np(state["lens"]), state["pool"], case["page"]
    seqs, heads, kv, hd = case["seqs"], case["heads"], case["kv"], case["hd"]
    q = _np(state["q"]).reshape(seqs, heads, hd)
    if "cos" in state:
        q = _turned(q, _np(state["turn"]), _np(state["cos"]), _np(state["sin"]), case["halves"], True)
    q, qs = (torch.from_numpy(a).cuda() for a in _int8(q))
    out = torch.zeros(seqs, heads, hd, dtype=torch.float64, device="cuda")
    mass = torch.zeros(pool["mass"].shape, dtype=torch.float64, device="cuda")
    for b in range(seqs):
        n = int(lens[b])
        if n == 0:
            continue
        ids = pool["table"][b, : -(-n // page)].long()
        for h in range(kv):
            at = (ids, h) if case["heads_first"] else (ids, slice(None), h)
            k, v = (_stored(pool[a][at].flatten(0, 1)[:n], pool[a + "p"][at].flatten(0, 1)[:n], hd) for a in ("k", "v"))
            g = slice(h * (heads // kv), (h + 1) * (heads // kv))
            p = torch.softmax((q[b, g] * qs[b, g]) @ k.T / math.sqrt(hd), -1)
            out[b, g] = p @ v
            new = torch.zeros(len(ids) * page, dtype=torch.float64, device="cuda")
            new[:n] = p.sum(0)
            mass[at] = new.reshape(len(ids), page)
    found = {"out": out.reshape(seqs, heads * hd)}
    if case["mass"]:
        found["mass"] = mass
    return found


def _exact_evict(state, case):
    lens, pool, page, kv, hd = _np(state["lens"]), state["pool"], case["page"], case["kv"], case["hd"]
    table, budget = _np(pool["table"]), case["budget"]
    mass, k, v = _np(pool["mass"]), pool["k"], pool["v"]
    kept = np.full((case["seqs"], kv, budget), -1, np.int64)
    back = {n: np.zeros((case["seqs"], budget, kv, hd)) for n in ("k", "v")}
    for b in range(case["seqs"]):
        n = int(lens[b])
        old = np.arange(n - min(n, case["recent"]))
        for h in range(kv):
            ids = table[b, np.arange(n) // page]
            where = (ids, h, np.arange(n) % page) if case["heads_first"] else (ids, np.arange(n) % page, h)
            choice = np.arange(n)
            if n > budget:
                m = mass[where][old]
                best = np.lexsort((old, -m))[: budget - case["recent"]]
                choice = np.concatenate((np.sort(old[best]), np.arange(n - case["recent"], n)))
            kept[b, h, : len(choice)] = choice
            spot = tuple(torch.from_numpy(w[choice]).cuda() if isinstance(w, np.ndarray) else w for w in where)
            for name, x in (("k", k), ("v", v)):
                back[name][b, : len(choice), h] = _np(_stored(x[spot], pool[name + "p"][spot], hd))
    rows = case["seqs"] * budget
    return {"k": back["k"].reshape(rows, -1), "v": back["v"].reshape(rows, -1), "kept": kept,
            "lens": np.minimum(lens, budget)}


def _exact_product(state, case):
    q, scale = _int8(_np(state["x"]))
    whole = torch.from_numpy(q).cuda() @ state["w"][:, : case["k"]].double().T
    y = whole * torch.from_numpy(scale).cuda() * state["ws"].double()
    return {"y": y + state["bias"].double() if case["bias"] else y}


def _exact_rope(state, case):
    pos = _np(state["pos"])
    live = pos >= 0
    x = _np(state["x"]).reshape(case["rows"], case["heads"], case["hd"])
    y = np.zeros_like(x)
    y[live] = _turned(x[live], pos[live], _np(state["cos"]), _np(state["sin"]), case["halves"], False)
    return {"y": y.reshape(case["rows"], -1)}


def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attention": _exact_attention, "evict": _exact_evict,
            "product": _exact_product}[case["op"]](state, case)
