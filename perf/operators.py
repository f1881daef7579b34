"""The serving operators over a paged int8 key/value cache, as cases to be timed and compared.

Four operators of one decode step of a server: new rows are rotated, quantised and written into the
pages of their sequences and can be read back ("append", "read"), one new token per sequence attends
over its pages ("attention"), and the next token of every row is sampled ("sample").

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
        # one sequence of a 0.5B-class model (2 kv heads of 64) takes its next token: pure latency
        dict(name="append_1x2x64", op="append", rows=1, seqs=1, kv=2, hd=64, page=16, context=513, rope=True,
             heads_first=False, padding=0),
        # one decode step of 64 sequences at context about 2048 (1B-class heads), each its own position
        dict(name="append_64x8x64", op="append", rows=64, seqs=64, kv=8, hd=64, page=32, context=2304, rope=True,
             heads_first=True, padding=0),
        # the prompts of four sequences of an 8B-class model written in one call, padding rows among them
        dict(name="append_16384x8x128", op="append", rows=16384, seqs=4, kv=8, hd=128, page=64, context=4352,
             rope=True, heads_first=False, padding=37),
        # a few odd rows read back (head size no power of two, pages of 7 positions)
        dict(name="read_333x3x80", op="read", rows=333, seqs=5, kv=3, hd=80, page=7, context=211,
             heads_first=False, padding=3),
        # the whole cache of two long sequences read back, to be moved or attended over elsewhere
        dict(name="read_32768x8x128", op="read", rows=32768, seqs=2, kv=8, hd=128, page=64, context=16512,
             heads_first=True, padding=0),
        # the smallest step: one short sequence, 14 query heads on 2 kv heads
        dict(name="attention_1x513_14x2x64", op="attention", seqs=1, longest=513, shortest=513, empty=0, heads=14,
             kv=2, hd=64, page=16, rope=True, heads_first=False),
        # a batch of equal sequences at context 2048 + 128
        dict(name="attention_64x2176_32x8x64", op="attention", seqs=64, longest=2176, shortest=2048, empty=0,
             heads=32, kv=8, hd=64, page=32, rope=True, heads_first=False),
        # ragged lengths from one token to 8192, and places of the batch that hold no sequence
        dict(name="attention_48xragged_32x8x128", op="attention", seqs=48, longest=8192, shortest=1, empty=3,
             heads=32, kv=8, hd=128, page=64, rope=False, heads_first=True),
        # one very long sequence: all the parallelism has to come from the cache's length
        dict(name="attention_1x131072_32x8x128", op="attention", seqs=1, longest=131072, shortest=131072, empty=0,
             heads=32, kv=8, hd=128, page=64, rope=True, heads_first=False),
        # one row over a 151,936-token vocabulary with every filter on
        dict(name="sample_1x151936", op="sample", rows=1, vocab=151936, top_k=50, filters="all"),
        # a batch whose rows ask for nucleus sampling alone: masses over the whole vocabulary
        dict(name="sample_64x128256_top_p", op="sample", rows=64, vocab=128256, top_k=0, filters="top_p"),
        # a large batch of rows with different settings (greedy, top-k, top-p, min-p, none)
        dict(name="sample_256x128256_mixed", op="sample", rows=256, vocab=128256, top_k=1000, filters="mixed"),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attention", "attention", "sample", "sample"])
    if op in ("append", "read"):
        hd = rng.choice([4 * rng.randint(4, 64), 64, 80, 96, 128, 256])
        kv = rng.randint(1, 16)
        rows = min(_log(rng, 1, 32768), (32768 * 8 * 128) // (kv * hd))
        rows = min(rows, 16384 * 8 * 128 // (kv * hd)) if op == "append" else rows
        seqs = rng.randint(1, min(rows, 64))
        case = dict(op=op, rows=rows, seqs=seqs, kv=kv, hd=hd, page=rng.choice([1, 7, 16, 32, 64, 128, 257]),
                    context=-(-rows // seqs) + rng.randint(0, 300), heads_first=rng.random() < 0.5,
                    padding=rng.choice([0, 0, rng.randint(0, rows // 4)]))
        if op == "append":
            case["rope"] = rng.random() < 0.5
        return case
    if op == "attention":
        hd = rng.choice([4 * rng.randint(4, 64), 64, 80, 96, 128, 256])
        kv, group = rng.randint(1, 8), rng.choice([1, 2, 4, 7, 8, 12, 16, 24])
        seqs = _log(rng, 1, 128)
        most = max(8, 131072 * 8 * 128 // (seqs * kv * hd))
        longest = _log(rng, 1, min(most, 131072, max(1, 40_000_000 // (seqs * kv * group))))
        return dict(op=op, seqs=seqs, longest=longest, shortest=rng.randint(1, longest),
                    empty=rng.choice([0, 0, rng.randint(0, seqs - 1)]), heads=kv * group, kv=kv, hd=hd,
                    page=rng.choice([1, 7, 16, 32, 64, 128, 257]), rope=rng.random() < 0.5,
                    heads_first=rng.random() < 0.5)
    vocab = _log(rng, 17, 160000)
    return dict(op=op, rows=min(_log(rng, 1, 256), max(1, 256 * 128256 // vocab)), vocab=vocab,
                top_k=_log(rng, 1, 4000), filters=rng.choice(["all", "top_k", "top_p", "min_p", "none", "mixed"]))


# ---------------------------------------------------------------------------------------------------
# Inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tables(positions, hd):
    """cos and sin [positions][hd / 2] of interleaved pairs, theta 5e5 (angles in 64 bits)."""
    j = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * 5e5 ** (-2.0 * j / hd)
    return angle.cos().float(), angle.sin().float()


def _pool(case, gen, filled):
    """A page pool with a quarter more pages than the sequences need, and a shuffled page table."""
    width = -(-(case["context"] if "context" in case else case["longest"]) // case["page"])
    seqs, page, kv, hd = case["seqs"], case["page"], case["kv"], case["hd"]
    pages = seqs * width + seqs * width // 4 + 1
    shape = (pages, kv, page) if case["heads_first"] else (pages, page, kv)
    pool = {"num_pages": pages, "page": page, "width": width, "heads_first": case["heads_first"]}
    for name in ("k", "v"):
        if filled:
            x = torch.empty(shape + (hd,), dtype=torch.int8, device="cuda")
            for a in x.split(max(1, (1 << 26) // (page * kv * hd))):
                a.copy_(torch.randn(a.shape, generator=gen, device="cuda").mul_(42).clamp_(-127, 127).round_())
            s = 0.01 + 0.02 * torch.rand(shape, generator=gen, device="cuda")
        else:
            x = torch.zeros(shape + (hd,), dtype=torch.int8, device="cuda")
            s = torch.zeros(shape, device="cuda")
        pool[name], pool[name + "s"] = x, s
    order = torch.randperm(pages, generator=gen, device="cuda")[: seqs * width]
    pool["table"] = order.to(torch.int32).reshape(seqs, width).contiguous()
    return pool


def _rows(case, gen):
    """Which (sequence, position) each row is: every sequence's last rows, and padding rows at random places."""
    rows, seqs = case["rows"], case["seqs"]
    i = torch.arange(rows, device="cuda")
    seq, k = i % seqs, i // seqs
    room = case["context"] - -(-rows // seqs)
    start = torch.randint(0, room + 1, (seqs,), generator=gen, device="cuda")
    pos = start[seq] + k
    order = torch.argsort(seq, stable=True)
    seq, pos = seq[order], pos[order]
    if case["padding"]:
        pos[torch.randperm(rows, generator=gen, device="cuda")[: case["padding"]]] = -1
    return seq.to(torch.int32), pos.to(torch.int32)


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": case}
    op = case["op"]
    if op in ("append", "read"):
        state["pool"] = _pool(case, gen, op == "read")
        state["seq"], state["pos"] = _rows(case, gen)
        width = case["kv"] * case["hd"]
        if op == "append":
            # the key and value columns of a fused projection's rows
            fused = torch.randn(case["rows"], 2 * width, generator=gen, device="cuda")
            state["k"], state["v"] = fused[:, :width], fused[:, width:]
            if case["rope"]:
                state["cos"], state["sin"] = _tables(case["context"], case["hd"])
        state["k_back"] = torch.zeros(case["rows"], width, device="cuda")
        state["v_back"] = torch.zeros(case["rows"], width, device="cuda")
    elif op == "attention":
        state["pool"] = _pool(case, gen, True)
        lens = torch.randint(case["shortest"], case["longest"] + 1, (case["seqs"],), generator=gen, device="cuda")
        lens[torch.randint(0, case["seqs"], (1,), generator=gen, device="cuda")] = case["longest"]
        if case["empty"]:
            lens[torch.randperm(case["seqs"], generator=gen, device="cuda")[: case["empty"]]] = 0
        state["lens"] = lens.to(torch.int32)
        width = case["heads"] * case["hd"]
        state["q"] = 2.0 * torch.randn(case["seqs"], width, generator=gen, device="cuda")
        state["out"] = torch.zeros(case["seqs"], width, device="cuda")
        if case["rope"]:
            state["cos"], state["sin"] = _tables(case["longest"], case["hd"])
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = 2.5 * torch.randn(rows, vocab, generator=gen, device="cuda")
        # some tokens stand out, as in a model's logits; some are forbidden
        count = min(vocab, 24)
        likely = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        likely = (likely + torch.arange(count, device="cuda") * (vocab // count)) % vocab
        logits.scatter_(1, likely, 8 + 6 * torch.rand(likely.shape, generator=gen, device="cuda"))
        banned = torch.randint(0, vocab, (rows, vocab // 64), generator=gen, device="cuda")
        logits.scatter_(1, banned, -math.inf)
        state["logits"] = logits
        uniform = lambda a, b: a + (b - a) * torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
        kind, f = torch.arange(rows, device="cuda") % 5, case["filters"]
        on = lambda name, k: f in ("all", name) or f == "mixed"  # noqa: E731
        mixed = lambda x, off, k: torch.where((kind == k) | (kind == 4), x, off) if f == "mixed" else x  # noqa: E731
        temperature = uniform(0.5, 1.3)
        state["temperature"] = torch.where(kind == 0, 0.0, temperature) if f == "mixed" else temperature
        if on("top_k", 1):
            state["top_k"] = mixed(torch.full((rows,), case["top_k"], device="cuda"), 0, 1).to(torch.int32)
        if on("top_p", 2):
            state["top_p"] = mixed(uniform(0.8, 0.98), 1.0, 2).contiguous()
        if on("min_p", 3):
            state["min_p"] = mixed(uniform(0.01, 0.1), 0.0, 3).contiguous()
        state["u"] = uniform(0.0, 1.0)
        state["ids"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        state["probs"] = torch.zeros(rows, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------
# The plain forms


def _slots(hd):
    """The slot of each rotated pair: the cache's order swaps pairs 2,3 and 4,5 of every full group of 8."""
    half = hd // 2
    order = [p + 2 if p % 8 in (2, 3) else p - 2 if p % 8 in (4, 5) else p for p in range(half - half % 8)]
    return order + list(range(half - half % 8, half))


def _rotate(x, pos, cos, sin):
    """x [rows, heads, hd] rotated by its row's position: two products, the second rounded, one fused sum."""
    hd = x.shape[-1]
    c, s = cos[pos][:, None].double(), sin[pos][:, None].double()
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    r0 = (a * c - (b * s).float().double()).float()
    r1 = (a * s + (b * c).float().double()).float()
    order = torch.tensor(_slots(hd), device=x.device)
    return torch.stack((r0[..., order], r1[..., order]), dim=-1).reshape(x.shape)


def _quantise(x):
    """Whole numbers in -127..127 (as floats) and one scale for each last axis."""
    amax = x.abs().amax(-1)
    c127 = torch.full_like(amax, 127.0)
    zero = torch.zeros_like(amax)
    inverse = torch.where(amax > 1e-8, c127 / amax, zero)
    scale = torch.where(amax > 1e-8, amax / c127, zero)
    return (x * inverse[..., None]).clamp(-127.0, 127.0).round(), scale


def _places(pool):
    """The pool's arrays as [pages, positions, kv heads, ...] whatever their order in memory."""
    names = ("k", "ks", "v", "vs")
    return [pool[n].transpose(1, 2) if pool["heads_first"] else pool[n] for n in names]


def _plain_append(state):
    case, pool = state["case"], state["pool"]
    live = state["pos"] >= 0
    seq, pos = state["seq"][live].long(), state["pos"][live].long()
    page, slot = pool["table"][seq, pos // pool["page"]].long(), pos % pool["page"]
    shape = (-1, case["kv"], case["hd"])
    k, v = state["k"][live].reshape(shape), state["v"][live].reshape(shape)
    if "cos" in state:
        k = _rotate(k, pos, state["cos"], state["sin"])
    pk, pks, pv, pvs = _places(pool)
    for x, to, scales in ((k, pk, pks), (v, pv, pvs)):
        q, s = _quantise(x)
        to[page, slot] = q.to(torch.int8)
        scales[page, slot] = s


def _plain_read(state):
    pool = state["pool"]
    live = state["pos"] >= 0
    seq, pos = state["seq"][live].long(), state["pos"][live].long()
    page, slot = pool["table"][seq, pos // pool["page"]].long(), pos % pool["page"]
    pk, pks, pv, pvs = _places(pool)
    for x, scales, back in ((pk, pks, "k_back"), (pv, pvs, "v_back")):
        state[back][live] = (x[page, slot].float() * scales[page, slot][..., None]).flatten(1)


def _plain_attention(state):
    case, pool, lens = state["case"], state["pool"], state["lens"].long()
    seqs, heads, kv, hd = case["seqs"], case["heads"], case["kv"], case["hd"]
    q = state["q"].reshape(seqs, heads, hd)
    if "cos" in state:
        q = _rotate(q, (lens - 1).clamp(min=0), state["cos"], state["sin"])
    q, qs = _quantise(q)
    at = torch.arange(case["longest"], device="cuda")
    page, slot = pool["table"][:, at // pool["page"]].long(), at % pool["page"]
    pk, pks, pv, pvs = _places(pool)
    k, v = (x[page, slot].permute(0, 2, 1, 3) for x in (pk, pv))  # [seqs, kv, positions, hd]
    ks, vs = (x[page, slot].permute(0, 2, 1)[:, :, None] for x in (pks, pvs))
    q, qs = q.reshape(seqs, kv, -1, hd), qs.reshape(seqs, kv, -1, 1)
    dots = q @ k.float().transpose(-1, -2)  # whole numbers below 2^24
    scores = dots * ((ks * qs) * (1.0 / math.sqrt(hd)))
    here = (at < lens[:, None])[:, None, None]
    scores = torch.where(here, scores, -math.inf)
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = (scores - m).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.where(here, p * vs, 0.0) @ v.float()
    state["out"].copy_(torch.where(total > 0, out / total, 0.0).reshape(seqs, -1))


def _plain_sample(state):
    """Masses in 64 bits: which token a draw falls on depends on sums next to a border."""
    logits, rows = state["logits"], state["case"]["rows"]
    vocab = logits.shape[1]
    l = logits.double()
    l = torch.where(l.isnan(), -math.inf, l)
    top = l.amax(-1, keepdim=True)
    t = state["temperature"].double()[:, None]
    greedy = ~(t > 0)
    z = torch.where(l == top, 0.0, (l - top) / torch.where(greedy, 1.0, t))
    w = torch.where(l == -math.inf, 0.0, z.exp())
    w = torch.where(w < 2.0 ** -40, 0.0, w)
    order = l.argsort(dim=-1, descending=True, stable=True)
    rank = torch.arange(vocab, device="cuda").expand(rows, -1)
    keep = torch.ones_like(rank, dtype=torch.bool)
    by_rank = w.gather(1, order)
    if "top_k" in state:
        k = state["top_k"].long()[:, None]
        keep &= (rank < k) | (k <= 0)
    if "top_p" in state:
        p = state["top_p"].double()[:, None]
        sums = torch.where(keep, by_rank, 0.0).cumsum(-1)
        before = torch.nn.functional.pad(sums[:, :-1], (1, 0))
        keep &= (before < p * sums[:, -1:]) | (p >= 1) | (rank == 0)
    if "min_p" in state:
        keep &= by_rank >= state["min_p"].double()[:, None].clamp(max=1.0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, by_rank, 0.0))
    reach = kept.cumsum(-1)
    total = reach[:, -1:]
    last = torch.where(kept > 0, rank, -1).amax(-1)
    pick = ((reach > state["u"].double()[:, None] * total).int() * (kept > 0).int()).argmax(-1)
    none = (reach <= state["u"].double()[:, None] * total).all(-1)
    pick = torch.where(none, last, pick)
    pick = torch.where(greedy[:, 0], order[:, 0], pick)
    prob = torch.where(greedy[:, 0], 1.0, kept.gather(1, pick[:, None])[:, 0] / total[:, 0])
    dead = top[:, 0] == -math.inf
    state["ids"].copy_(torch.where(dead, -1, pick))
    state["probs"].copy_(torch.where(dead, 0.0, prob))


# ---------------------------------------------------------------------------------------------------
# The framework's calls


def _kv_pages(pool):
    from jieyu_b200 import _capi
    k, s = pool["k"], pool["ks"]
    a, b = (2, 1) if pool["heads_first"] else (1, 2)
    return _capi.KVPages(k.data_ptr(), s.data_ptr(), pool["v"].data_ptr(), pool["vs"].data_ptr(), pool["num_pages"],
                         pool["page"], k.stride(0), k.stride(a), k.stride(b), s.stride(0), s.stride(a), s.stride(b))


def _at(state, name):
    return state[name].data_ptr() if name in state else None


def _calls(state):
    """The calls of one pass as (function, arguments before the stream): a program makes them once per buffer set."""
    import ctypes

    from jieyu_b200 import _capi
    lib, case = _capi.load(), state["case"]
    if case["op"] == "sample":
        logits = state["logits"]
        return [(lib.jyc_sample_batch,
                 (logits.data_ptr(), logits.stride(0), case["rows"], case["vocab"], _at(state, "temperature"),
                  _at(state, "top_k"), _at(state, "top_p"), _at(state, "min_p"), _at(state, "u"), _at(state, "ids"),
                  _at(state, "probs")))]
    pool = state["pool"]
    state["pages"] = _kv_pages(pool)
    pages = ctypes.byref(state["pages"])
    table = (pool["table"].data_ptr(), pool["width"], case["seqs"])
    rope = (_at(state, "cos"), _at(state, "sin"), state["cos"].shape[0] if "cos" in state else 0)
    if case["op"] == "attention":
        need = lib.jyc_attention_paged_q8_workspace(case["seqs"], case["heads"], case["kv"], case["hd"])
        state["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        return [(lib.jyc_attention_paged_q8,
                 (_at(state, "q"), state["q"].stride(0), _at(state, "out"), state["out"].stride(0), case["heads"],
                  case["kv"], case["hd"], _at(state, "lens")) + table + rope
                 + (pages, state["workspace"].data_ptr(), need))]
    rows = (case["rows"], case["kv"], case["hd"], _at(state, "seq"), _at(state, "pos")) + table
    read = (lib.jyc_kv_read_paged_q8,
            (_at(state, "k_back"), _at(state, "v_back"), state["k_back"].stride(0)) + rows + (pages,))
    if case["op"] == "read":
        return [read]
    return [(lib.jyc_kv_append_paged_q8,
             (_at(state, "k"), _at(state, "v"), state["k"].stride(0)) + rows + rope + (pages,)), read]


def run(state):
    """One pass. What an append writes is held in 8 bits: the rows come back as the values they stand for,
    through the read operator, which is part of the pass."""
    op = state["case"]["op"]
    if own:
        if "calls" not in state:
            state["calls"] = _calls(state)
        stream = torch.cuda.current_stream().cuda_stream
        for call, arguments in state["calls"]:
            status = call(*arguments, stream)
            if status < 0:
                raise RuntimeError("status %d" % status)
    elif op == "append":
        _plain_append(state)
        _plain_read(state)
    elif op == "read":
        _plain_read(state)
    elif op == "attention":
        _plain_attention(state)
    else:
        _plain_sample(state)
    if op == "attention":
        return {"out": state["out"]}
    if op == "sample":
        return {"ids": state["ids"], "probs": state["probs"]}
    return {"k": state["k_back"], "v": state["v_back"]}


# ---------------------------------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    kv, hd = case["kv"], case["hd"]
    if op == "attention":
        live = case["seqs"] - case["empty"]
        tokens = live * (case["longest"] + case["shortest"]) / 2
        q_out = 8 * case["seqs"] * case["heads"] * hd
        return {"bytes": tokens * kv * (2 * hd + 8) + 4 * tokens / case["page"] + q_out,
                "flops": 4 * tokens * case["heads"] * hd}
    rows = max(1, case["rows"] - case["padding"])
    in_cache, in_floats = rows * kv * (2 * hd + 8), rows * kv * hd * 8
    if op == "read":
        return {"bytes": in_cache + in_floats + 8 * case["rows"], "flops": 2 * rows * kv * hd}
    tables = 4 * hd * min(rows, case["context"]) if case["rope"] else 0
    return {"bytes": 2 * (in_cache + in_floats) + tables + 16 * case["rows"], "flops": 12 * rows * kv * hd}


# ---------------------------------------------------------------------------------------------------
# The definitions in 64 bits, with numpy. The cache's whole numbers and scales are 32-bit roundings by
# definition (inverse 127 / amax, product, scale amax / 127), made here by rounding 64-bit results.


def _f32(x):
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def _np(x):
    x = x.cpu().numpy()
    return x.astype(np.float64) if x.dtype == np.float32 else x.astype(np.int64)


def _turned(x, pos, cos, sin):
    out = np.empty_like(x)
    half = x.shape[-1] // 2
    for p in range(half):
        to = p
        if p - p % 8 + 8 <= half:
            to = p - p % 8 + [0, 1, 4, 5, 2, 3, 6, 7][p % 8]
        c, s = cos[pos, p][:, None], sin[pos, p][:, None]
        a, b = x[:, :, 2 * p], x[:, :, 2 * p + 1]
        out[:, :, 2 * to] = _f32(a * c - _f32(b * s))
        out[:, :, 2 * to + 1] = _f32(a * s + _f32(b * c))
    return out


def _eight(x):
    amax = np.max(np.abs(x), axis=-1, keepdims=True)
    tiny = amax <= np.float64(np.float32(1e-8))
    safe = np.where(tiny, 1.0, amax)
    inverse, scale = np.where(tiny, 0.0, _f32(127.0 / safe)), np.where(tiny, 0.0, _f32(safe / 127.0))
    return np.rint(np.clip(_f32(x * inverse), -127, 127)), scale


def _exact_rows(state, case):
    pos, seq, pool = _np(state["pos"]), _np(state["seq"]), state["pool"]
    rows, kv, hd = case["rows"], case["kv"], case["hd"]
    live = pos >= 0
    found = {}
    for name in ("k", "v"):
        back = np.zeros((rows, kv, hd))
        if case["op"] == "append":
            x = _np(state[name]).reshape(rows, kv, hd)[live]
            if name == "k" and case["rope"]:
                x = _turned(x, pos[live], _np(state["cos"]), _np(state["sin"]))
            q, s = _eight(x)
            back[live] = q * s
        else:
            x, s = pool[name].cpu().numpy(), _np(pool[name + "s"])
            page = _np(pool["table"])[seq[live], pos[live] // case["page"]]
            slot = pos[live] % case["page"]
            if case["heads_first"]:
                back[live] = x[page, :, slot] * s[page, :, slot][..., None]
            else:
                back[live] = x[page, slot] * s[page, slot][..., None]
        found[name] = back.reshape(rows, kv * hd)
    return found


def _exact_attention(state, case):
    lens, table, pool = _np(state["lens"]), state["pool"]["table"].long(), state["pool"]
    seqs, heads, kv, hd, page = case["seqs"], case["heads"], case["kv"], case["hd"], case["page"]
    q = _np(state["q"]).reshape(seqs, heads, hd)
    if case["rope"]:
        q = _turned(q, np.maximum(lens - 1, 0), _np(state["cos"]), _np(state["sin"]))
    q, qs = (torch.from_numpy(a).cuda() for a in _eight(q))
    out = torch.zeros(seqs, heads, hd, dtype=torch.float64, device="cuda")
    for b in range(seqs):
        n = int(lens[b])
        if n == 0:
            continue
        need = table[b, : -(-n // page)]
        for h in range(kv):
            if case["heads_first"]:
                k, v, ks, vs = (pool[a][need, h].flatten(0, 1)[:n].double() for a in ("k", "v", "ks", "vs"))
            else:
                k, v, ks, vs = (pool[a][need, :, h].flatten(0, 1)[:n].double() for a in ("k", "v", "ks", "vs"))
            g = slice(h * (heads // kv), (h + 1) * (heads // kv))
            score = (q[b, g] * qs[b, g]) @ (k * ks[:, None]).T / math.sqrt(hd)
            out[b, g] = torch.softmax(score, -1) @ (v * vs[:, None])
    return {"out": out.reshape(seqs, heads * hd)}


def _exact_sample(state, case):
    rows = case["rows"]
    logits, u, temperature = _np(state["logits"]), _np(state["u"]), _np(state["temperature"])
    setting = {n: _np(state[n]) if n in state else None for n in ("top_k", "top_p", "min_p")}
    ids, probs = np.zeros(rows, np.int64), np.zeros(rows)
    for r in range(rows):
        l = np.where(np.isnan(logits[r]), -np.inf, logits[r])
        best = int(np.argmax(l))
        if l[best] == -np.inf:
            ids[r], probs[r] = -1, 0.0
            continue
        if not temperature[r] > 0:
            ids[r], probs[r] = best, 1.0
            continue
        w = np.where(l == l[best], 1.0, np.exp((np.where(l == l[best], 0.0, l - l[best])) / temperature[r]))
        w[w < 2.0 ** -40] = 0.0
        chosen = np.argsort(-l, kind="stable")
        if setting["top_k"] is not None and setting["top_k"][r] > 0:
            chosen = chosen[: setting["top_k"][r]]
        if setting["top_p"] is not None and setting["top_p"][r] < 1:
            sums = np.cumsum(w[chosen])
            chosen = chosen[: 1 + int(np.searchsorted(sums, setting["top_p"][r] * sums[-1], side="left"))]
        if setting["min_p"] is not None:
            chosen = chosen[w[chosen] >= min(1.0, setting["min_p"][r])]
        chosen = np.sort(chosen[w[chosen] > 0])
        sums = np.cumsum(w[chosen])
        at = min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), chosen.size - 1)
        ids[r], probs[r] = chosen[at], w[chosen[at]] / sums[-1]
    return {"ids": ids, "probs": probs}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("append", "read"):
        return _exact_rows(state, case)
    return _exact_attention(state, case) if case["op"] == "attention" else _exact_sample(state, case)
