"""The operators on token ids that stand on either side of a model, as cases that can be timed: the embedding lookup and its
gradient, the page tables and slot maps of a paged cache, and the verification of drafted tokens.

`own` chooses between the plain forms (elementary torch operations) and the calls into libl3hip.so; both take the same
state.  Every size is a case's own: the vocabulary of 128,256 entries is the tokenizer's, the rest is generic."""
import math

import torch

own = False

VOCAB = 128256
_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODE = {"f32": 0, "f16": 1, "bf16": 2}     # L3_F32, L3_F16, L3_BF16
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one step of a serving batch: the last token of 64 requests
        _embed("embed decode", n=64, rows=VOCAB, dim=4096, table="bf16", out="bf16", scale=1.0),
        # the prompts of a serving step, or one micro-batch of training, with the scaling some models put on the lookup
        _embed("embed prompts", n=16384, rows=VOCAB, dim=4096, table="bf16", out="bf16", scale=64.0),
        # a small model with an odd width, 32-bit weights under 16-bit activations
        _embed("embed odd width", n=3001, rows=50001, dim=1001, table="f32", out="bf16", scale=0.5),
        # fine-tuning: a few hundred tokens onto 32-bit main gradients
        _grad("grad small step", n=512, rows=VOCAB, dim=2048, grad="bf16", table="f32", scale=1.0, accumulate=True),
        # a large training step: 65,536 tokens onto 32-bit main gradients
        _grad("grad large step", n=65536, rows=VOCAB, dim=4096, grad="bf16", table="f32", scale=1.0, accumulate=True),
        # a gradient written whole, odd sizes, 16 bits throughout
        _grad("grad whole odd", n=5003, rows=50001, dim=1001, grad="f16", table="f16", scale=0.5, accumulate=False),
        # one token for each of 256 requests that are under way
        _slots("slots decode", seqs=256, page=16, pages=1 << 17, most=512, tokens=256, new_lo=1, new_hi=1, old_hi=8000, tight=False),
        # 2,048 prompts at once, of one to 4,096 tokens, cut off where the step's room for tokens ends
        _slots("slots prompts", seqs=2048, page=16, pages=1 << 17, most=512, tokens=1 << 20, new_lo=1, new_hi=4096, old_hi=0, tight=False),
        # drafts that were not accepted leave 256 requests a few tokens shorter
        _trim("trim after drafts", seqs=256, page=16, pages=1 << 17, most=512, old_hi=8000, back=8, finished=0.0),
        # a third of 2,048 requests has ended
        _trim("trim finished", seqs=2048, page=16, pages=1 << 19, most=512, old_hi=8000, back=0, finished=0.33),
        # a single request with four drafted tokens, where latency is what counts
        _verify("verify one", seqs=1, draft=4, vocab=VOCAB, dtype="bf16", with_q=True),
        # a serving batch: 128 requests, up to eight drafted tokens each
        _verify("verify batch", seqs=128, draft=8, vocab=VOCAB, dtype="f32", with_q=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["embed", "grad", "slots", "trim", "verify"])
    scale = rng.choice([1.0, 0.5, 64.0, 45.25])
    if kind == "embed":
        n, dim = log(1, 16384), log(64, 4096)
        dim = dim if rng.random() < 0.4 else max(64, dim // 64 * 64)
        table = rng.choice(["bf16", "f16", "f32"])
        return _embed(None, n=n, rows=log(1000, VOCAB), dim=dim, table=table, out=rng.choice([table, "bf16"]), scale=scale)
    if kind == "grad":
        n, dim = log(1, 65536), log(64, 4096)
        dim = dim if rng.random() < 0.4 else max(64, dim // 64 * 64)
        grad, acc = rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.6
        table = "f32" if acc else rng.choice([grad, "f32"])
        return _grad(None, n=n if grad != "f32" else max(1, n // 2), rows=log(1000, VOCAB), dim=dim, grad=grad, table=table,
                     scale=scale, accumulate=acc)
    page = rng.choice([16, 32, 64, 128])
    if kind == "slots":
        hi, seqs = log(1, 4096), log(1, 2048)
        return _slots(None, seqs=seqs, page=page, pages=1 << 17, most=8192 // page, tokens=log(seqs, max(seqs, min(1 << 20, seqs * hi // 2))),
                      new_lo=rng.choice([0, 1]), new_hi=hi, old_hi=rng.choice([0, 8192 - hi]), tight=rng.random() < 0.3)
    if kind == "trim":
        return _trim(None, seqs=log(1, 2048), page=page, pages=1 << 19, most=8192 // page, old_hi=8192, back=rng.randint(0, 8),
                     finished=rng.choice([0.0, 0.1, 0.5]))
    return _verify(None, seqs=log(1, 128), draft=rng.randint(1, 8), vocab=rng.choice([VOCAB, log(1000, VOCAB)]),
                   dtype=rng.choice(["f32", "bf16", "f16"]), with_q=rng.random() < 0.7)


def _case(op, name, **k):
    return dict(k, op=op, **({"name": name} if name else {}))


def _embed(name, **k):
    return _case("embed", name, **k)


def _grad(name, **k):
    return _case("grad", name, **k)


def _slots(name, **k):
    return _case("slots", name, **k)


def _trim(name, **k):
    return _case("trim", name, **k)


def _verify(name, **k):
    return _case("verify", name, **k)


# ---- inputs -------------------------------------------------------------------------------------------------------
def _ids(n, rows, g):
    """Token ids as text has them: the more frequent the lower (frequency ~ 1 / rank), one in fifty a pad (-1)."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    ids = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1).int()
    ids[torch.rand(n, device="cuda", generator=g) < 0.02] = -1
    return ids


def _rand(shape, dtype, g):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(_DTYPE[dtype])


def _held_pages(seqs, most, pages, held, g):
    """A pool of pages in no order: the first of them in the tables of the requests, the others free."""
    order = torch.randperm(pages, device="cuda", generator=g).int()
    first = torch.cumsum(held.long(), 0) - held
    j = torch.arange(most, device="cuda")
    at = (first[:, None] + j).clamp_(max=pages - 1)
    table = torch.where(j < held[:, None], order[at], torch.full_like(order[at], -1))
    used = held.sum()
    free = torch.where(torch.arange(pages, device="cuda") < pages - used, order.flip(0), torch.full_like(order, -1))
    return table, free, (pages - used).int().reshape(1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": dict(case)}
    op = case["op"]
    if op == "embed":
        s["ids"] = _ids(case["n"], case["rows"], g)
        s["table"] = _rand((case["rows"], case["dim"]), case["table"], g)
        s["out"] = torch.empty(case["n"], case["dim"], device="cuda", dtype=_DTYPE[case["out"]])
    elif op == "grad":
        s["ids"] = _ids(case["n"], case["rows"], g)
        s["grad"] = _rand((case["n"], case["dim"]), case["grad"], g)
        s["table"] = _rand((case["rows"], case["dim"]), case["table"], g)   # gradients of earlier micro-batches, or stale ones
        work = 64 * case["n"] + case["n"] * case["dim"] + (4 << 20)
        s["work"] = torch.empty(work, device="cuda", dtype=torch.uint8)
    elif op in ("slots", "trim"):
        n, page, most = case["seqs"], case["page"], case["most"]
        limit = min(most * page, case["pages"] * page // (2 * n))            # the tables never hold more than half of the pool
        old = torch.randint(0, case["old_hi"] + 1, (n,), device="cuda", generator=g).clamp_(max=limit)
        held = (old + page - 1) // page
        s["table"], s["free"], s["n_free"] = _held_pages(n, most, case["pages"], held, g)
        s["length"], s["held"] = old.int(), held.int()
        s["length_out"], s["held_out"], s["n_free_out"] = (torch.empty_like(s[k]) for k in ("length", "held", "n_free"))
        s["status"] = torch.empty(1, device="cuda", dtype=torch.int32)
        s["work"] = torch.empty(64 * n + 65536, device="cuda", dtype=torch.uint8)
        if op == "slots":
            u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
            new = torch.exp(u * math.log(case["new_hi"] - case["new_lo"] + 1.0)).long() - 1 + case["new_lo"]
            s["off"] = torch.cat([new.new_zeros(1), torch.cumsum(new, 0).clamp_(max=case["tokens"])])
            new = s["off"][1:] - s["off"][:-1]
            s["slots"] = torch.full((case["tokens"],), -7, device="cuda", dtype=torch.int64)   # what is behind the last token stays
            s["pos"] = torch.full((case["tokens"],), -7, device="cuda", dtype=torch.int32)
            if case["tight"]:                                                # the pool runs short within the batch
                s["n_free"] = torch.minimum(s["n_free"], (new.sum() // (2 * page)).int().reshape(1))
        else:
            back = torch.randint(0, case["back"] + 1, (n,), device="cuda", generator=g)
            ended = torch.rand(n, device="cuda", generator=g) < case["finished"]
            keep = torch.where(ended, torch.zeros_like(old), (old - back).clamp_(min=0))
            if case["finished"]:
                keep = torch.where(ended, keep, torch.full_like(keep, -1))   # the others are not looked at
            s["keep"] = keep.int()
    else:
        n, most, vocab, t = case["seqs"], case["draft"], case["vocab"], _DTYPE[case["dtype"]]
        k = torch.randint(0, most + 1, (n,), device="cuda", generator=g)
        k[0] = most
        s["off"] = torch.cat([k.new_zeros(1), torch.cumsum(k, 0)])
        total = int(s["off"][-1])
        logit = torch.randn(total + n, vocab, device="cuda", generator=g).mul_(3.0)
        s["target"] = torch.softmax(logit, -1).to(t)
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), k)
        row = torch.arange(total, device="cuda") + seq                        # the target's row of each drafted token
        near = logit[row].add_(torch.randn(total, vocab, device="cuda", generator=g).mul_(0.7))
        del logit
        q = torch.softmax(near, -1)
        del near
        s["q"] = q.to(t) if case["with_q"] else None
        # the drafted tokens: drawn from the draft's probabilities, or its most likely ones
        if case["with_q"]:
            cut = torch.rand(total, 1, device="cuda", generator=g, dtype=torch.float64)
            c = torch.cumsum(q.double(), -1)
            s["draft"] = (c <= cut * c[:, -1:]).sum(-1).clamp_(max=vocab - 1).int()
        else:
            s["draft"] = q.argmax(-1).int()
        s["u_accept"] = torch.rand(total, device="cuda", generator=g)
        s["u_draw"] = torch.rand(n, device="cuda", generator=g)
        s["out"] = torch.empty(n, most + 1, device="cuda", dtype=torch.int32)
        s["accepted"] = torch.empty(n, device="cuda", dtype=torch.int32)
        s["work"] = torch.empty(4096 * n + 65536, device="cuda", dtype=torch.uint8)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------
_context = None


def _ctx():
    """The tokenizer's context, made once by a program that uses it."""
    global _context
    if _context is None:
        from tokenizer_amd import capi
        _context = capi.Context(device=0)
    return _context


def run(s):
    return {"embed": _run_embed, "grad": _run_grad, "slots": _run_slots, "trim": _run_trim, "verify": _run_verify}[s["case"]["op"]](s)


def _run_embed(s):
    c = s["case"]
    ids, table = s["ids"], s["table"]
    if own:
        _ctx().embed(ids.data_ptr(), c["n"], table.data_ptr(), _CODE[c["table"]], c["rows"], c["dim"], c["dim"], s["out"].data_ptr(),
                     _CODE[c["out"]], c["dim"], c["scale"])
        return s["out"]
    there = ((ids >= 0) & (ids < c["rows"]))[:, None]
    rows = table[ids.clamp(0, c["rows"] - 1).long()].float() * c["scale"]
    return torch.where(there, rows, torch.zeros_like(rows)).to(_DTYPE[c["out"]])


def _run_grad(s):
    c = s["case"]
    ids, grad, table = s["ids"], s["grad"], s["table"]
    if own:
        _ctx().embed_grad(ids.data_ptr(), c["n"], grad.data_ptr(), _CODE[c["grad"]], c["dim"], c["rows"], c["dim"], table.data_ptr(),
                          _CODE[c["table"]], c["dim"], s["work"].data_ptr(), s["work"].numel(), c["scale"], c["accumulate"])
        return table
    there = ((ids >= 0) & (ids < c["rows"]))[:, None]
    rows = grad.float() * c["scale"]
    rows = torch.where(there, rows, torch.zeros_like(rows))
    at = ids.clamp(0, c["rows"] - 1).long()
    if c["accumulate"] and c["table"] == "f32":
        return table.index_add_(0, at, rows)
    total = torch.zeros(c["rows"], c["dim"], device=table.device).index_add_(0, at, rows)
    return table.copy_(total + table.float() if c["accumulate"] else total)


def _run_slots(s):
    c = s["case"]
    n, page, most, pages = c["seqs"], c["page"], c["most"], c["pages"]
    off, length, held, free, n_free = s["off"], s["length"], s["held"], s["free"], s["n_free"]
    if own:
        _ctx().cache_slots(off.data_ptr(), n, length.data_ptr(), held.data_ptr(), page, pages, s["table"].data_ptr(), most, most,
                           free.data_ptr(), n_free.data_ptr(), s["length_out"].data_ptr(), s["held_out"].data_ptr(),
                           s["n_free_out"].data_ptr(), s["slots"].data_ptr(), s["pos"].data_ptr(), c["tokens"], s["status"].data_ptr(),
                           s["work"].data_ptr(), s["work"].numel())
        return {"table": s["table"], "length": s["length_out"], "held": s["held_out"], "n_free": s["n_free_out"], "slots": s["slots"],
                "pos": s["pos"], "status": s["status"]}
    new = off[1:] - off[:-1]
    old, have, left = length.long(), held.long(), n_free.long()
    fits = old + new <= most * page
    need = torch.where(fits, ((old + new + page - 1) // page - have).clamp_(min=0), torch.zeros_like(old))
    end = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (end <= left))
    j = torch.arange(most, device=off.device)
    fresh = (j >= have[:, None]) & (j < (have + need)[:, None]) & served[:, None]
    at = (left - 1 - (end - need)[:, None] - (j - have[:, None])).clamp_(0, pages - 1)
    table = torch.where(fresh, free[at], s["table"])
    t = torch.arange(c["tokens"], device=off.device)
    there = t < off[-1]
    seq = (torch.searchsorted(off, t, right=True) - 1).clamp_(max=n - 1)
    pos = old[seq] + t - off[seq]
    slot = table[seq, (pos // page).clamp_(max=most - 1)].long() * page + pos % page
    slot, pos = (torch.where(served[seq], x, torch.full_like(x, -1)) for x in (slot, pos))
    taken = torch.where(served, need, torch.zeros_like(need))
    status = (~fits).any().int() * 2 + (fits & ~served).any().int()
    return {"table": table, "length": torch.where(served, old + new, old).int(), "held": (have + taken).int(),
            "n_free": (left - taken.sum()).int(), "slots": torch.where(there, slot, s["slots"]),
            "pos": torch.where(there, pos.int(), s["pos"]), "status": status.reshape(1)}


def _run_trim(s):
    c = s["case"]
    n, page, most, pages = c["seqs"], c["page"], c["most"], c["pages"]
    keep, length, held, free, n_free = s["keep"], s["length"], s["held"], s["free"], s["n_free"]
    if own:
        _ctx().cache_trim(keep.data_ptr(), n, length.data_ptr(), held.data_ptr(), page, pages, s["table"].data_ptr(), most, most,
                          free.data_ptr(), n_free.data_ptr(), s["length_out"].data_ptr(), s["held_out"].data_ptr(),
                          s["n_free_out"].data_ptr(), s["status"].data_ptr(), s["work"].data_ptr(), s["work"].numel())
        return {"free": free, "length": s["length_out"], "held": s["held_out"], "n_free": s["n_free_out"], "status": s["status"]}
    old, have, left = length.long(), held.long(), n_free.long()
    asked = keep >= 0
    now = torch.where(asked, torch.minimum(keep.long(), old), old)
    stay = torch.where(asked, (now + page - 1) // page, have)
    give = have - stay
    end = torch.cumsum(give, 0)
    j = torch.arange(most, device=keep.device)
    goes = (j >= stay[:, None]) & (j < have[:, None])
    at = torch.where(goes, left + (end - give)[:, None] + j - stay[:, None], torch.full_like(goes, pages, dtype=torch.long))
    grown = torch.cat([free, free.new_zeros(1)])
    grown[at.reshape(-1)] = s["table"].reshape(-1)      # what stays lands behind the pool
    return {"free": grown[:pages], "length": now.int(), "held": stay.int(), "n_free": (left + end[-1]).int(),
            "status": torch.zeros(1, device=keep.device, dtype=torch.int32)}


def _run_verify(s):
    c = s["case"]
    n, most, vocab = c["seqs"], c["draft"], c["vocab"]
    off, draft, target, q = s["off"], s["draft"], s["target"], s["q"]
    if own:
        _ctx().verify_draft(draft.data_ptr(), off.data_ptr(), n, draft.numel(), most, target.data_ptr(), _CODE[c["dtype"]], vocab,
                            q.data_ptr() if q is not None else None, vocab, vocab, s["u_accept"].data_ptr(), s["u_draw"].data_ptr(),
                            s["out"].data_ptr(), s["accepted"].data_ptr(), s["work"].data_ptr(), s["work"].numel())
        return {"tokens": s["out"], "accepted": s["accepted"]}
    k = off[1:] - off[:-1]
    j = torch.arange(most, device=off.device)
    there = j < k[:, None]
    seq = torch.arange(n, device=off.device)
    at = (off[:-1, None] + j).clamp_(max=draft.numel() - 1)
    d = draft[at].long()
    p = target[(at + seq[:, None]).clamp_(max=target.shape[0] - 1), d].double()
    qd = q[at, d].double() if q is not None else torch.ones_like(p)
    accepted = torch.cumprod((there & (s["u_accept"][at].double() * qd < p)).long(), 1).sum(1)
    weight = target[off[:-1] + accepted + seq].double()
    at = (off[:-1] + accepted).clamp_(max=draft.numel() - 1)
    if q is not None:
        rest = (weight - q[at].double()).clamp_(min=0.0)
    else:
        rest = weight.scatter(1, draft[at].long()[:, None], 0.0)
    stopped = (accepted < k)[:, None]
    weight = torch.where(stopped & (rest.sum(-1, keepdim=True) > 0), rest, weight)
    sums = torch.cumsum(weight, -1)
    token = (sums <= s["u_draw"].double()[:, None] * sums[:, -1:]).sum(-1).clamp_(max=vocab - 1)
    spot = torch.arange(most + 1, device=off.device)
    drafts = torch.cat([d, d.new_zeros(n, 1)], 1)
    out = torch.where(spot < accepted[:, None], drafts, torch.where(spot == accepted[:, None], token[:, None], torch.full_like(drafts, -1)))
    return {"tokens": out.int(), "accepted": accepted.int()}


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def _distinct(n, rows):
    """How many different ids n draws of _ids give, about: rank r (from 1) has the share log(1 + 1/r) / log(rows + 1)."""
    total, lo = 0.0, 1
    while lo <= rows:                     # ranks in bands, so that the sum stays short
        hi = min(rows + 1, max(lo + 1, lo * 9 // 8))
        share = math.log(hi / lo) / (hi - lo) / math.log(rows + 1.0)
        total += (hi - lo) * -math.expm1(0.98 * n * math.log1p(-share))
        lo = hi
    return total


def work(case):
    op = case["op"]
    if op == "embed":
        u = _distinct(case["n"], case["rows"])
        return {"bytes": 4 * case["n"] + case["dim"] * (u * _SIZE[case["table"]] + case["n"] * _SIZE[case["out"]]),
                "flops": case["n"] * case["dim"]}
    if op == "grad":
        u = _distinct(case["n"], case["rows"])
        rows = 2 * u if case["accumulate"] else case["rows"]
        return {"bytes": 4 * case["n"] + case["dim"] * (0.98 * case["n"] * _SIZE[case["grad"]] + rows * _SIZE[case["table"]]),
                "flops": 2 * case["n"] * case["dim"]}
    n, page = case.get("seqs"), case.get("page")
    if op == "slots":
        span = case["new_hi"] - case["new_lo"] + 1.0
        new = min(case["tokens"], n * (case["new_lo"] + ((span - 1.0) / math.log(span) - 1.0 if span > 1 else 0.0)))
        return {"bytes": 24 * n + 8 + 12 * new + 8 * max(1.0, new / page), "flops": 4 * new + 8 * n}
    if op == "trim":
        mean = min(case["old_hi"], case["most"] * page, case["pages"] * page // (2 * n)) / 2
        gone = n * (case["finished"] * mean / page + case["back"] / 2 / page)
        return {"bytes": 20 * n + 8 * gone, "flops": 8 * n + gone}
    arrays = 2 if case["with_q"] else 1
    return {"bytes": n * (case["vocab"] * _SIZE[case["dtype"]] * arrays + 16 * case["draft"] + 24), "flops": n * case["vocab"] * (1 + arrays)}


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------
def exact(case, seed):
    """The lookup and its gradient from sums over sorted ids; the other operators answer with whole numbers."""
    if case["op"] == "embed":
        s = prepare(case, seed)
        pad = torch.cat([s["table"], s["table"].new_zeros(1, case["dim"])]).double()
        return pad[torch.where(s["ids"] < 0, case["rows"], s["ids"]).long()].mul_(case["scale"])
    if case["op"] == "grad":
        s = prepare(case, seed)
        ids, order = torch.sort(torch.where(s["ids"] < 0, case["rows"], s["ids"]).long(), stable=True)
        sums = torch.cumsum(s["grad"].double()[order], 0)
        sums = torch.cat([sums.new_zeros(1, case["dim"]), sums])
        ends = torch.searchsorted(ids, torch.arange(case["rows"] + 1, device=ids.device))
        total = (sums[ends[1:]] - sums[ends[:-1]]).mul_(case["scale"])
        return total.add_(s["table"].double()) if case["accumulate"] else total
    return None
