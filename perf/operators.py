"""The operators of a decoder's memory, as cases that can be timed and compared.

A paged key-value cache (appending to it, attention of one new token over it, eviction from
it by accumulated attention weight) and linear attention with a decay for each head.  `run`
computes an operator in elementary torch operations, or, where `own` is true, with the
framework's kernels on the same device memory.
"""
import math
import random

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------- cases --
def listed():
    return [
        # one short conversation on an encoder-sized model (12 heads of 64): latency counts
        dict(name="attend one short row", op="attend", batch=1, heads=12, kv_heads=12, dim=64,
             page=16, min_len=128, max_len=128, weights=False, mask=False),
        # a serving batch of grouped heads whose left-padded prompts are masked
        dict(name="attend ragged masked batch", op="attend", batch=16, heads=32, kv_heads=8, dim=128,
             page=16, min_len=1, max_len=2048, weights=True, mask=True),
        # one document of 100 thousand tokens: few rows, a long axis
        dict(name="attend one long row", op="attend", batch=1, heads=32, kv_heads=8, dim=128,
             page=64, min_len=100003, max_len=100003, weights=False, mask=False),
        # a full machine: 64 rows up to 8192 tokens, weights kept for eviction
        dict(name="attend large batch", op="attend", batch=64, heads=32, kv_heads=4, dim=64,
             page=32, min_len=257, max_len=8192, weights=True, mask=False),
        # one decoding step of a batch
        dict(name="append one token", op="append", batch=32, kv_heads=8, dim=128, page=16,
             tokens=1, min_count=1, min_len=0, max_len=2047),
        # prompts of differing lengths, padded to the longest
        dict(name="append prompts", op="append", batch=8, kv_heads=8, dim=64, page=16,
             tokens=2048, min_count=1, min_len=0, max_len=0),
        # steady state: one token too many in every row
        dict(name="evict one slot", op="evict", batch=32, kv_heads=8, dim=64, page=16,
             min_len=1025, max_len=1025, budget=1024, recent=256, positions=True),
        # prompts cut down to a budget before decoding begins
        dict(name="evict after prompts", op="evict", batch=16, kv_heads=8, dim=128, page=16,
             min_len=777, max_len=8192, budget=2048, recent=512, positions=False),
        # one token of one row
        dict(name="linear one token", op="linear", batch=1, heads=12, seq=1, min_len=1,
             dim=64, dim_v=64, state=True),
        # one token of a serving batch: the states are what is read and written
        dict(name="linear batch of tokens", op="linear", batch=64, heads=16, seq=1, min_len=1,
             dim=128, dim_v=128, state=True),
        # prompts of differing lengths
        dict(name="linear prompts", op="linear", batch=4, heads=12, seq=2047, min_len=1000,
             dim=64, dim_v=64, state=False),
        # long documents that continue from a state
        dict(name="linear long rows", op="linear", batch=2, heads=16, seq=16384, min_len=16384,
             dim=128, dim_v=128, state=True),
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "evict", "linear", "linear"])
    while True:
        dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 192])
        page = rng.choice([8, 16, 16, 32, 64, 128])
        if op == "attend":
            kv = rng.choice([1, 2, 4, 8, 12, 16])
            group = rng.choice([1, 1, 2, 3, 4, 7, 8])
            hi = _log(rng, 1, 100000)
            case = dict(op=op, batch=_log(rng, 1, 64), heads=kv * group, kv_heads=kv, dim=dim,
                        page=page, min_len=rng.choice([hi, _log(rng, 1, hi)]), max_len=hi,
                        weights=rng.random() < 0.5, mask=rng.random() < 0.25)
        elif op == "append":
            t = rng.choice([1, _log(rng, 2, 4096)])
            hi = rng.choice([0, _log(rng, 1, 8192)])
            case = dict(op=op, batch=_log(rng, 1, 64), kv_heads=rng.choice([1, 2, 4, 8, 12, 16]),
                        dim=dim, page=page, tokens=t, min_count=rng.choice([0, t]),
                        min_len=rng.choice([0, hi]), max_len=hi)
        elif op == "evict":
            hi = _log(rng, 16, 32768)
            budget = max(1, int(hi * rng.uniform(0.05, 1.0)))
            case = dict(op=op, batch=_log(rng, 1, 32), kv_heads=rng.choice([1, 2, 4, 8, 12, 16]),
                        dim=dim, page=page, min_len=rng.choice([hi, _log(rng, 1, hi)]), max_len=hi,
                        budget=budget, recent=rng.choice([0, budget // 4, budget // 2]),
                        positions=rng.random() < 0.5)
        else:
            s = rng.choice([1, _log(rng, 2, 16384), _log(rng, 64, 16384)])
            case = dict(op=op, batch=_log(rng, 1, 64), heads=rng.choice([1, 2, 4, 8, 12, 16, 32]),
                        seq=s, min_len=rng.choice([s, _log(rng, 1, s)]), dim=rng.choice([16, 32, 64, 96, 128]),
                        dim_v=rng.choice([32, 64, 64, 100, 128]), state=s == 1 or rng.random() < 0.5)
        if _cost(case) <= max(_cost(c) for c in listed() if c["op"] == op):
            return case


def _spread(lo, hi, n, salt):
    """n whole numbers from lo to hi, hi among them, the same for the same case."""
    r = random.Random(lo * 7919 + hi * 104729 + n * 31 + salt)
    v = [hi] + [r.randint(lo, hi) for _ in range(n - 1)]
    r.shuffle(v)
    return v


def _lengths(case):
    if case["op"] == "linear":
        return _spread(case["min_len"], case["seq"], case["batch"], 1)
    return _spread(case["min_len"], case["max_len"], case["batch"], 1)


def _counts(case):
    return _spread(case["min_count"], case["tokens"], case["batch"], 2)


def _capacity(case):
    """Slots of a row: whole pages."""
    most = case["max_len"] + (case["tokens"] if case["op"] == "append" else 0)
    return max(1, -(-most // case["page"])) * case["page"]


# ------------------------------------------------------------------------- inputs --
def _pools(case, g, filled):
    """Key and value pools, and a table that spreads the rows' pages over them; entries that
    a row does not need are -1."""
    p = case["page"]
    need = [-(-n // p) for n in filled]
    total = sum(need) + 3
    order = torch.randperm(total, generator=torch.Generator().manual_seed(int(g.initial_seed()) % (1 << 31)))
    table = torch.full((case["batch"], _capacity(case) // p), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (total, case["kv_heads"], p, case["dim"])
    return (torch.randn(shape, device=DEV, generator=g), torch.randn(shape, device=DEV, generator=g),
            table.to(DEV))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lengths = _lengths(case)
    s = {"case": case, "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV)}
    rnd = lambda *shape: torch.randn(shape, device=DEV, generator=g)  # noqa: E731
    b = case["batch"]
    if case["op"] == "linear":
        h, n, dk, dv = case["heads"], case["seq"], case["dim"], case["dim_v"]
        s["q"], s["k"], s["v"] = rnd(b, h, n, dk), rnd(b, h, n, dk) / math.sqrt(dk), rnd(b, h, n, dv)
        # decays of 1 - 2^-5 to 1 - 2^-12, evenly in the exponent, as retention layers set them
        e = torch.linspace(5.0, 12.0, h, dtype=torch.float64)
        s["log_decay"] = torch.log1p(-torch.exp2(-e)).to(torch.float32).to(DEV)
        s["state"] = rnd(b, h, dk, dv) if case["state"] else None
        s["scale"] = 1.0 / math.sqrt(dk)
        return s
    if case["op"] == "append":
        counts = _counts(case)
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
        s["k_cache"], s["v_cache"], s["table"] = _pools(case, g, [n + c for n, c in zip(lengths, counts)])
        s["k"] = rnd(b, case["kv_heads"], case["tokens"], case["dim"])
        s["v"] = rnd(b, case["kv_heads"], case["tokens"], case["dim"])
        return s
    s["k_cache"], s["v_cache"], s["table"] = _pools(case, g, lengths)
    cap = _capacity(case)
    slot = torch.arange(cap, device=DEV)
    inside = slot < s["lengths"][:, None]
    if case["op"] == "attend":
        s["q"] = rnd(b, case["heads"], 1, case["dim"])
        s["scale"] = 1.0 / math.sqrt(case["dim"])
        s["mask"] = None
        if case["mask"]:  # the first tenth of a row is padding
            hidden = slot < (s["lengths"][:, None] // 10)
            s["mask"] = torch.where(hidden, -math.inf, 0.0).to(torch.float32)
        s["weights"] = None
        if case["weights"]:
            w = torch.rand(b, case["kv_heads"], cap, device=DEV, generator=g)
            s["weights"] = torch.where(inside[:, None], w, 0.0)
        return s
    # accumulated weights: a few heavy slots, many light ones, and new ones that have none yet
    w = torch.exp(2.0 * rnd(b, case["kv_heads"], cap) - 6.0)
    new = slot >= s["lengths"][:, None] - case["recent"] // 2
    s["weights"] = torch.where((inside & ~new)[:, None], w, 0.0)
    s["positions"] = s["total"] = None
    if case["positions"]:
        # earlier evictions left the slots below 7/8 of the row in an order of their own
        old = (s["lengths"] * 7 // 8)[:, None, None]
        key = torch.where(slot < old, torch.rand(b, case["kv_heads"], cap, device=DEV, generator=g), 2.0)
        at = torch.argsort(torch.argsort(key, dim=-1), dim=-1)
        s["positions"] = torch.where(slot < old, 2 * at, -1).to(torch.int32)
        s["total"] = (s["lengths"] * 2 + 1).to(torch.int32)
    return s


# -------------------------------------------------------------------- plain forms --
def _rows(pool, table):
    """[batch, kv_heads, capacity, dim] of a pool's pages; places without a page hold page 0."""
    x = pool[table.long().clamp(min=0)]                      # [B, pages, Hkv, P, D]
    b, n, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, n * p, d)


def _attend(s):
    case = s["case"]
    b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    inside = (torch.arange(_capacity(case), device=DEV) < s["lengths"][:, None])[:, None, None]
    zero = torch.zeros((), device=DEV)
    k = torch.where(inside.transpose(2, 3), _rows(s["k_cache"], s["table"]), zero)
    v = torch.where(inside.transpose(2, 3), _rows(s["v_cache"], s["table"]), zero)
    x = torch.matmul(s["q"].reshape(b, kv, h // kv, d), k.transpose(2, 3)) * s["scale"]
    if s["mask"] is not None:
        x = x + s["mask"][:, None, None]
    x = torch.where(inside, x, -math.inf)
    m = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    z = e.double().sum(dim=-1, keepdim=True)
    p = torch.where(z > 0, e / z, 0.0).float()
    # a long row is summed in pieces
    n = p.shape[-1]
    step = 512 if n % 512 == 0 else case["page"]
    o = torch.matmul(p.reshape(b, kv, h // kv, n // step, step).transpose(2, 3),
                     v.reshape(b, kv, n // step, step, d)).double().sum(dim=2).float()
    out = {"out": o.reshape(b, 1, h, d)}
    if s["weights"] is not None:
        out["weights"] = torch.where(inside[:, :, 0], s["weights"] + p.sum(dim=2), 0.0)
    return out


def _append(s):
    case = s["case"]
    p = case["page"]
    live = torch.arange(case["tokens"], device=DEV) < s["counts"][:, None]
    row, t = live.nonzero(as_tuple=True)
    at = s["lengths"].long()[row] + t
    page = s["table"].long()[row, at // p]
    s["k_cache"][page, :, at % p] = s["k"][row, :, t]
    s["v_cache"][page, :, at % p] = s["v"][row, :, t]
    return {"lengths": s["lengths"] + s["counts"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _evict(s):
    case = s["case"]
    p, cap = case["page"], _capacity(case)
    slot = torch.arange(cap, device=DEV)
    n = s["lengths"].long()[:, None, None]
    m = n.clamp(max=case["budget"])
    total = n if s["total"] is None else s["total"].long()[:, None, None]
    pos = (total - (n - slot)).expand(s["weights"].shape)
    if s["positions"] is not None:
        pos = torch.where(s["positions"] >= 0, s["positions"].long(), pos)
    key = torch.where(pos >= total - case["recent"], math.inf, s["weights"])
    key = torch.where(slot < n, key, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(order, dtype=torch.bool).scatter_(2, order, (slot < m).expand(order.shape))
    hole, tail = (slot < m) & ~keep, (slot >= m) & keep
    # the r-th hole takes the r-th kept slot behind the budget
    tails = torch.sort(torch.where(tail, slot, cap), dim=-1).values
    rank = (torch.cumsum(hole, dim=-1) - 1).clamp(min=0)
    src = torch.where(hole, torch.gather(tails, 2, rank), slot)
    src = torch.where(slot < m, src, 0)
    b, h, to = hole.nonzero(as_tuple=True)
    frm = src[b, h, to]
    table = s["table"].long()
    for pool in (s["k_cache"], s["v_cache"]):
        pool[table[b, to // p], h, to % p] = pool[table[b, frm // p], h, frm % p]
    left = slot < m
    return {"weights": torch.where(left, torch.gather(s["weights"], 2, src), 0.0),
            "positions": torch.where(left, torch.gather(pos, 2, src), -1).to(torch.int32),
            "lengths": m[:, 0, 0].to(torch.int32),
            "kept": torch.where(left, src, -1)[:, :, :case["budget"]].to(torch.int32).contiguous(),
            "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _linear(s):
    case = s["case"]
    b, h, n, dk, dv = case["batch"], case["heads"], case["seq"], case["dim"], case["dim_v"]
    c = min(64, n)
    chunks = -(-n // c)
    pad = chunks * c - n
    g = s["log_decay"].double()[:, None, None]
    live = torch.arange(n, device=DEV) < s["lengths"][:, None]
    zero = torch.zeros((), device=DEV)
    cut = lambda x: torch.nn.functional.pad(  # noqa: E731
        torch.where(live[:, None, :, None], x, zero), (0, 0, 0, pad)).reshape(b, h, chunks, c, x.shape[-1])
    q, k, v = cut(s["q"]), cut(s["k"]), cut(s["v"])
    t = torch.arange(c, device=DEV, dtype=torch.float64)
    ago = t[:, None] - t[None, :]
    inner = torch.where(ago >= 0, torch.exp(g * ago.clamp(min=0)), 0.0).float()[:, None]      # [H, 1, C, C]
    o = torch.matmul(torch.matmul(q, k.transpose(3, 4)) * inner, v)
    # what each chunk adds, as it stands at the chunk's end, and the state before each chunk
    add = torch.matmul((k * torch.exp(g * (c - 1 - t)[:, None]).float()[:, None]).transpose(3, 4), v)
    i = torch.arange(chunks + 1, device=DEV, dtype=torch.float64)
    far = i[:, None] - 1 - i[None, :chunks]
    carry = torch.where(far >= 0, torch.exp(g * c * far.clamp(min=0)), 0.0).float()           # [H, chunks + 1, chunks]
    state = torch.matmul(carry, add.reshape(b, h, chunks, dk * dv))
    if s["state"] is not None:
        state = state + torch.exp(g * c * i[:, None]).float() * s["state"].reshape(b, h, 1, dk * dv)
    state = state.reshape(b, h, chunks + 1, dk, dv)
    o = o + torch.matmul(q * torch.exp(g * (t + 1)[:, None]).float()[:, None], state[:, :, :chunks])
    o = (o * s["scale"]).reshape(b, h, chunks * c, dv)[:, :, :n].transpose(1, 2).contiguous()
    # tokens behind a row's end added nothing, but decayed what was there: from the state in front of the
    # row's last chunk instead
    at = s["lengths"].long() // c
    rest = (s["lengths"].long() - at * c).double()[:, None, None, None]
    last = state[torch.arange(b, device=DEV), :, at]
    at = at.clamp(max=chunks - 1)
    rows = torch.arange(b, device=DEV)
    w = torch.where(t < rest[..., 0], torch.exp(g[None, :, 0] * (rest[..., 0] - 1 - t).clamp(min=0)), 0.0).float()
    tail = torch.matmul((k[rows, :, at] * w[..., None]).transpose(2, 3), v[rows, :, at])
    return {"out": o, "state": torch.exp(g[None] * rest).float() * last + tail}


# ------------------------------------------------------------ the framework's calls --
class _Held(dict):
    """The framework's tensors over device memory that a program keeps from step to step;
    disposed with the program's state."""

    def __del__(self):
        for t in self.values():
            if t is not None:
                t.dispose()


def _handle(tf, s, name):
    held = s.setdefault("held", _Held())
    if name not in held:
        held[name] = tf.tensor(s[name]) if s[name] is not None else None
    return held[name]


def _run_own(s):
    import tfjs_b200
    from tfjs_b200 import ops as tf
    tfjs_b200.ENGINE.ready()
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    new, out = [], {}

    def fresh(name):
        """A tensor that is new in every step."""
        new.append(tf.tensor(s[name], stream=stream))
        return new[-1]

    if case["op"] == "linear":
        o, state = tf.linear_attention(fresh("q"), fresh("k"), fresh("v"), _handle(tf, s, "log_decay"),
                                       _handle(tf, s, "state"), s["scale"], _handle(tf, s, "lengths"))
        out = {"out": o, "state": state}
    else:
        pools = [_handle(tf, s, name) for name in ("k_cache", "v_cache")]
        table, lengths = _handle(tf, s, "table"), _handle(tf, s, "lengths")
        if case["op"] == "append":
            out["lengths"] = tf.paged_cache_append(*pools, fresh("k"), fresh("v"), table, lengths,
                                                   _handle(tf, s, "counts"))
        elif case["op"] == "attend":
            got = tf.paged_attention(fresh("q"), *pools, table, lengths, s["scale"], _handle(tf, s, "mask"),
                                     _handle(tf, s, "weights"))
            if case["weights"]:
                out["out"], out["weights"] = got
            else:
                out["out"] = got
        else:
            out["weights"], out["positions"], out["lengths"], out["kept"] = tf.paged_cache_evict(
                *pools, _handle(tf, s, "weights"), table, lengths, case["budget"], case["recent"],
                _handle(tf, s, "positions"), _handle(tf, s, "total"))
    result = {name: torch.as_tensor(t.dataToGPU(stream), device=DEV) for name, t in out.items()}
    for t in new + list(out.values()):
        t.dispose()
    if case["op"] in ("append", "evict"):
        result["k_cache"], result["v_cache"] = s["k_cache"], s["v_cache"]
    return result


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "append": _append, "evict": _evict, "linear": _linear}[state["case"]["op"]](state)


def work(case):
    op, n = case["op"], _lengths(case)
    d, b = case["dim"], case["batch"]
    if op == "linear":
        tokens, dv = sum(n) * case["heads"], case["dim_v"]
        states = (2 if case["state"] else 1) * b * case["heads"] * d * dv
        # outputs behind a row's end are written, as zeros
        return {"bytes": 4.0 * (tokens * (2 * d + dv) + b * case["heads"] * case["seq"] * dv + states),
                "flops": 4.0 * tokens * d * dv}
    kv, table = case["kv_heads"], 4.0 * sum(-(-v // case["page"]) for v in n)
    if op == "append":
        new = sum(_counts(case)) * kv * d
        return {"bytes": 4.0 * 4 * new + 12.0 * b, "flops": 0.0}
    cap = _capacity(case)
    if op == "attend":
        extra = (sum(n) * kv + b * kv * cap if case["weights"] else 0) + (sum(n) if case["mask"] else 0)
        return {"bytes": 4.0 * (2 * sum(n) * kv * d + 2 * b * case["heads"] * d + extra) + table,
                "flops": 4.0 * sum(n) * case["heads"] * d}
    moved = 0.0
    for v in n:  # slots kept behind the budget: the protected ones, and their share of the rest
        m = min(v, case["budget"])
        r = min(case["recent"], m)
        if v > m:
            moved += min(r, v - m) + (m - r) * max(0, v - r - m) / (v - r)
    read = sum(n) * kv * (2 if case["positions"] else 1)
    return {"bytes": 4.0 * (read + b * kv * (2 * cap + case["budget"]) + 4 * moved * kv * d) + table, "flops": 0.0}


# ------------------------------------------------------- the definitions in 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict,
            "linear": _exact_linear}[case["op"]](s, case)


def _exact_attend(s, case):
    out, weights = [], []
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(s["lengths"].tolist()):
        j = torch.arange(n, device=DEV)
        page = s["table"][b].long()[j // case["page"]]
        k, v = (s[x][page, :, j % case["page"]].double().repeat_interleave(group, dim=1)
                for x in ("k_cache", "v_cache"))                       # [n, H, D]
        a = torch.einsum("hd,nhd->hn", s["q"][b, :, 0].double(), k) * s["scale"]
        if s["mask"] is not None:
            a = a + s["mask"][b, :n].double()
        p = torch.softmax(a, dim=-1)
        out.append(torch.einsum("hn,nhd->hd", p, v)[None])
        if s["weights"] is not None:
            w = torch.zeros_like(s["weights"][b], dtype=torch.float64)
            w[:, :n] = s["weights"][b, :, :n].double() + p.reshape(-1, group, n).sum(dim=1)
            weights.append(w)
    return {"out": torch.stack(out), **({"weights": torch.stack(weights)} if weights else {})}


def _exact_append(s, case):
    for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
        pages, t, at = s["table"][b].tolist(), 0, n
        while t < c:                                                   # page by page
            page, off = pages[at // case["page"]], at % case["page"]
            few = min(case["page"] - off, c - t)
            s["k_cache"][page, :, off:off + few] = s["k"][b, :, t:t + few]
            s["v_cache"][page, :, off:off + few] = s["v"][b, :, t:t + few]
            t, at = t + few, at + few
    return {"lengths": s["lengths"] + s["counts"], "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}


def _exact_evict(s, case):
    """Weights, row by row; the whole outputs have to be equal in any case."""
    if sum(_lengths(case)) * case["kv_heads"] > 3e6:
        return None
    kept_weights = torch.zeros_like(s["weights"], dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        m = min(n, case["budget"])
        total = n if s["total"] is None else int(s["total"][b])
        for h in range(case["kv_heads"]):
            w = s["weights"][b, h, :n].tolist()
            pos = [total - n + j for j in range(n)]
            if s["positions"] is not None:
                pos = [x if x >= 0 else y for x, y in zip(s["positions"][b, h, :n].tolist(), pos)]
            by = sorted(range(n), key=lambda j: (pos[j] < total - case["recent"], -w[j] if pos[j] < total - case["recent"] else 0, j))
            keep = set(by[:m])
            late = iter(sorted(j for j in keep if j >= m))
            row = [w[j] if j in keep else w[next(late)] for j in range(m)]
            kept_weights[b, h, :m] = torch.tensor(row, dtype=torch.float64)
    return {"weights": kept_weights, "positions": None, "lengths": None, "kept": None, "k_cache": None, "v_cache": None}


def _exact_linear(s, case):
    b, h, n, dk, dv = case["batch"], case["heads"], case["seq"], case["dim"], case["dim_v"]
    if n * b * h * dk * dv > 1.5e11:
        return None
    decay = torch.exp(s["log_decay"].double())[None, :, None, None]
    state = s["state"].double() if s["state"] is not None else torch.zeros(b, h, dk, dv, dtype=torch.float64, device=DEV)
    out = torch.zeros(b, n, h, dv, dtype=torch.float64, device=DEV)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    for t in range(n):                                                 # the recurrence, token by token
        live = (t < s["lengths"])[:, None, None, None]
        state = torch.where(live, decay * state + k[:, :, t, :, None] * v[:, :, t, None, :], state)
        o = torch.matmul(q[:, :, t, None], state)[:, :, 0] * s["scale"]
        out[:, t] = torch.where(live[..., 0], o, 0.0)
    return {"out": out, "state": state}
