"""The cache operators of tree verification and of a bounded cache, as a serving loop calls them.

A step of speculative decoding scores a tree of drafted tokens against the cache (``sdpa_tree``), walks the
greedy path through it (``tree_accept``) and commits the accepted rows (``kv_append``).  A cache of bounded size
accumulates the attention weight every slot receives (``attn_mass``) and drops the slots with the least of it
(``kv_evict``).  ``run`` makes one of these calls, as the framework's kernel where ``own`` is true and as
elementary torch operations otherwise.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    head = dict(h=32, hk=8, d=128, dtype="bf16")            # the attention block of the 8B decoder
    return [
        # one sequence, a short context and eight candidates: the latency of a chat's first steps
        dict(name="tree one sequence", op="tree", n=1, l=8, s=600, used=517, **head),
        # a serving batch of ragged contexts, an odd number of candidates
        dict(name="tree batch", op="tree", n=16, l=27, s=4096, used=4001, **head),
        # long documents, a wide tree
        dict(name="tree long", op="tree", n=2, l=64, s=65536, used=65000, **dict(head, dtype="f16")),
        # one accepted token of one sequence and layer
        dict(name="append one token", op="append", layers=1, n=1, l=1, s=2048, used=1023, **head),
        # every layer of the decoder at once after a batch was verified
        dict(name="append all layers", op="append", layers=32, n=16, l=27, s=640, used=600, **head),
        # the walk through one small tree, and through the largest trees of a large batch
        dict(name="accept one sequence", op="accept", n=1, l=8, shared=True),
        dict(name="accept batch", op="accept", n=256, l=255, shared=False),
        # a decode step of a batch with long contexts: every key is read once for one token
        dict(name="mass decode", op="mass", n=8, l=1, s=16384, used=16001, causal=True, **head),
        # an observation window at the end of a prompt
        dict(name="mass window", op="mass", n=4, l=64, s=8191, used=8191, causal=True, **dict(head, dtype="f16")),
        # a whole prompt
        dict(name="mass prompt", op="mass", n=1, l=8192, s=8192, used=8192, causal=True, **head),
        # one layer of one sequence a little over its budget
        dict(name="evict one sequence", op="evict", layers=1, n=1, s=1200, used=1111, budget=1024, sinks=4, recent=64, **head),
        # half of a long cache in several layers of a batch
        dict(name="evict layers", op="evict", layers=8, n=8, s=16384, used=16384, budget=8192, sinks=4, recent=1024, **head),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "append", "accept", "mass", "mass", "evict"])
    if op == "accept":
        return dict(op=op, n=_log(rng, 1, 256), l=_log(rng, 1, 255), shared=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    hk = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 7, 8])
    d = rng.choice([64, 128, 128, 128, 80, 96]) if dtype != "f32" else rng.choice([64, 128])
    case = dict(op=op, h=hk * g, hk=hk, d=d, dtype=dtype)
    if op == "tree":
        l = _log(rng, 1, 64)
        n = _log(rng, 1, 16)
        # fp32 caches stay small: they are the form for checking a model
        s = _log(rng, 64, max(64, min(65536, (65536 * 2 if dtype != "f32" else 4096) // n)))
        case.update(n=n, l=l, s=s, used=max(1, s - rng.randrange(0, 1 + s // 3)))
    elif op == "append":
        layers, l = _log(rng, 1, 32), _log(rng, 1, 64)
        n = _log(rng, 1, 16)
        s = _log(rng, 2 * l + 1, 640)
        case.update(layers=layers, n=n, l=l, s=s, used=rng.randrange(0, s - l + 1))
    elif op == "mass":
        n, causal = _log(rng, 1, 8), rng.random() < 0.8
        s = _log(rng, 64, (131072 if dtype != "f32" else 8192) // n)
        l = rng.choice([1, _log(rng, 1, 64), _log(rng, 64, 4096) if dtype != "f32" else 64])
        l = max(1, min(l, s, (1 << 28) // max(1, s * n * hk * g)))
        case.update(n=n, l=l, s=s, used=max(l, s - rng.randrange(0, 1 + s // 3)), causal=causal)
    else:
        layers, n = _log(rng, 1, 8), _log(rng, 1, 8)
        s = _log(rng, 64, 16384)
        used = max(40, s - rng.randrange(0, 1 + s // 3))
        budget = rng.randrange(used // 4, used)
        recent = rng.randrange(0, budget // 4 + 1)
        case.update(layers=layers, n=n, s=s, used=used, budget=budget, sinks=rng.randrange(0, 5), recent=recent)
    return case


def _lens(case):
    """Ragged key counts: the first sequence holds `used` keys, the others fewer (the last of five or more none)."""
    n, used = case["n"], case["used"]
    least = case["l"] if case["op"] == "mass" else 0
    lens = [max(least, used - (i * 389) % (used // 2 + 1)) for i in range(n)]
    if n >= 5 and case["op"] == "tree":
        lens[-1] = 0
    return lens


def _counts(case):
    """Accepted rows per sequence: a few of those drafted."""
    return [min(case["l"], 1 + (3 * i) % 7) for i in range(case["n"])]


def _tree_parents(n, l, g):
    """Random trees: node i hangs below one of the nodes before it, more often below a recent one."""
    i = torch.arange(l, device="cuda").expand(n, l)
    u = torch.rand(n, l, generator=g, device="cuda")
    parents = (i - 1 - (u * u * i).long()).clamp_(min=0)
    parents[:, 0] = -1
    return parents


def _ancestors(parents):
    """bool [n, l, l]: node j is node i or one of its ancestors."""
    l = parents.shape[1]
    eye = torch.eye(l, device=parents.device)
    step = (torch.arange(l, device=parents.device) == parents[:, :, None]).float()
    # a node comes after its parent, so 1 + step + step^2 + ... is the inverse of a unit triangle; its entries are 0 and 1
    return torch.linalg.solve_triangular(eye - step, eye.expand_as(step), upper=False, unitriangular=True) > 0.5


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, n = case["op"], case["n"]
    st = {"case": case}
    if op == "accept":
        l = case["l"]
        st["parents"] = _tree_parents(1 if case["shared"] else n, l, g)
        st["target"] = torch.randint(0, 128256, (n, l), generator=g, device="cuda")
        # three of four drafted tokens are what the model would have said
        said = st["target"].gather(1, st["parents"].clamp(min=0).expand(n, l))
        right = torch.rand(n, l, generator=g, device="cuda") < 0.75
        st["draft"] = torch.where(right, said, torch.randint(0, 128256, (n, l), generator=g, device="cuda"))
        return st
    h, hk, d, s, dt = case["h"], case["hk"], case["d"], case["s"], _DT[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    layers = case.get("layers", 1)
    st["kv_lens"] = torch.tensor(_lens(case), device="cuda", dtype=torch.int64)
    st["K"] = rand(layers * n, hk, s, d)
    if op in ("tree", "append"):
        l = case["l"]
        st["V"] = rand(layers * n, hk, s, d)
        # q, k and v rows as the packed projection leaves them: (rows, (h + 2 hk) d)
        w = (h + 2 * hk) * d
        qkv = rand(layers * n * l, w)
        at = lambda heads, first: qkv.as_strided((layers * n, heads, l, d), (l * w, d, w, 1), first * d)  # noqa: E731
        st["Q"], st["Kd"], st["Vd"] = at(h, 0), at(hk, h), at(hk, h + hk)
    if op == "tree":
        st["mask"] = _ancestors(_tree_parents(n, case["l"], g))
    if op == "append":
        counts = _counts(case)
        st["counts"] = torch.tensor(counts, device="cuda", dtype=torch.int64)
        path = torch.rand(n, l, generator=g, device="cuda").argsort(1)[:, :max(counts)].sort(1).values
        st["path"] = torch.full((n, l), -1, device="cuda", dtype=torch.int64)
        st["path"][:, :max(counts)] = path
        st["pos"] = torch.randint(0, s, (layers * n, hk, s), generator=g, device="cuda", dtype=torch.int32)
        st["next_pos"] = st["kv_lens"] + 11
        st["mass"] = torch.rand(layers * n, hk, s, generator=g, device="cuda")
    if op == "mass":
        l, lens = case["l"], _lens(case)
        st["Q"] = rand(n, l, h, d).transpose(1, 2)
        # what a few calls like this one have left before it
        st["mass"] = torch.rand(n, hk, s, generator=g, device="cuda") * (4.0 * l * (h // hk) / case["used"])
        # the log-sum-exp that the attention call before this one left, to within what random scores make of it
        seen = torch.tensor(lens, device="cuda", dtype=torch.float32)[:, None]
        if case["causal"]:
            seen = seen - l + 1 + torch.arange(l, device="cuda", dtype=torch.float32)
        st["lse"] = (seen.log() + 0.5)[:, None, :] + 0.05 * torch.randn(n, h, l, generator=g, device="cuda")
        st["lse"] = st["lse"].contiguous()
    if op == "evict":
        st["V"] = rand(layers * n, hk, s, d)
        # attention weight falls off over several powers of two, as it does in a trained model
        st["mass"] = torch.exp(2.0 * torch.randn(layers * n, hk, s, generator=g, device="cuda"))
        st["pos"] = torch.arange(s, device="cuda", dtype=torch.int32).expand(layers * n, hk, s).contiguous()
        st["next_pos"] = st["kv_lens"].clone()
    return st


_kuiops = None


def _ffi():
    global _kuiops
    if _kuiops is None:
        from kuillm_b200.kuipy import _ffi as mod
        _kuiops = mod
    return _kuiops


def run(state):
    op = state["case"]["op"]
    if own:
        f = _ffi()
        if op == "tree":
            return f.sdpa_tree(state["Q"], state["K"], state["V"], state["kv_lens"], state["Kd"], state["Vd"], state["mask"])
        if op == "accept":
            return f.tree_accept(state["parents"], state["draft"], state["target"])
        if op == "append":
            lens = f.kv_append(state["K"], state["V"], state["kv_lens"], state["Kd"], state["Vd"], path=state["path"],
                               counts=state["counts"], pos=state["pos"], next_pos=state["next_pos"], mass=state["mass"])
            return lens, state["K"], state["V"], state["pos"], state["mass"]
        if op == "mass":
            return f.attn_mass(state["Q"], state["K"], state["lse"], kv_lens=state["kv_lens"],
                               is_causal=state["case"]["causal"], mass=state["mass"])
        c = state["case"]
        lens, mass, pos, src = f.kv_evict(state["K"], state["V"], state["mass"], state["kv_lens"], c["budget"], pos=state["pos"],
                                          next_pos=state["next_pos"], sinks=c["sinks"], recent=c["recent"])
        return lens, mass, pos, src, state["K"], state["V"]
    return {"tree": _plain_tree, "accept": _plain_accept, "append": _plain_append, "mass": _plain_mass, "evict": _plain_evict}[op](state)


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _plain_tree(st):
    q, k, v = st["Q"].float(), st["K"].float(), st["V"].float()
    n, h, l, d = q.shape
    hk, s = k.shape[1], k.shape[2]
    g = h // hk
    k = torch.cat([k, st["Kd"].float()], 2)
    v = torch.cat([v, st["Vd"].float()], 2)
    seen = torch.cat([(torch.arange(s, device=q.device) < st["kv_lens"][:, None])[:, None, :].expand(n, l, s), st["mask"]], 2)
    x = torch.matmul(q.reshape(n, hk, g * l, d), k.transpose(2, 3)).reshape(n, hk, g, l, s + l) / math.sqrt(d)
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(w.reshape(n, hk, g * l, s + l), v).reshape(n, h, l, d)
    lse = (top + total.log()).reshape(n, h, l)
    return out.to(st["Q"].dtype), lse


def _plain_accept(st):
    draft, target = st["draft"], st["target"]
    n, l = draft.shape
    parents = st["parents"].expand(n, l)
    ok = draft == target.gather(1, parents.clamp(min=0))
    ok = torch.cat([torch.ones_like(ok[:, :1]), ok[:, 1:]], 1)
    index = torch.arange(l, device=draft.device)
    over = _ancestors(parents)
    depth = over.sum(2)
    good = (over & ~ok[:, None, :]).sum(2) == 0                                   # every node on the way was said
    count = torch.where(good, depth, torch.zeros_like(depth))
    most = count.amax(1, keepdim=True)
    best = torch.where(count == most, index, l).amin(1)
    on = over[torch.arange(n, device=draft.device), best]                         # [n, l]
    place = torch.where(on, on.long().cumsum(1) - 1, l)                           # ancestors have smaller indices
    path = torch.full((n, l + 1), -1, device=draft.device, dtype=torch.int64)
    path.scatter_(1, place, index.expand(n, l))
    return torch.where(index < most, path[:, :l], torch.full_like(path[:, :l], -1)), most[:, 0], target.gather(1, best[:, None])[:, 0]


def _plain_append(st):
    K, V, lens, counts, path = st["K"], st["V"], st["kv_lens"], st["counts"], st["path"]
    rows, hk, s, d = K.shape
    n, l = path.shape
    per = rows // n
    t = torch.arange(l, device=K.device)
    live = t < counts[:, None]                                                    # [n, l]
    b, tt = torch.where(live)
    slot = lens[b] + tt
    row = (torch.arange(per, device=K.device)[:, None] * n + b).reshape(-1)       # [per * accepted]
    slot, src = slot.repeat(per), path[b, tt].repeat(per)
    K[row, :, slot] = st["Kd"][row, :, src]
    V[row, :, slot] = st["Vd"][row, :, src]
    st["pos"][row, :, slot] = (st["next_pos"][b] + tt).to(torch.int32).repeat(per)[:, None]
    st["mass"][row, :, slot] = 0.0
    return lens + counts, K, V, st["pos"], st["mass"]


def _plain_mass(st):
    c = st["case"]
    q, k = st["Q"].float(), st["K"].float()
    n, h, l, d = q.shape
    hk, s = k.shape[1], k.shape[2]
    g = h // hk
    x = torch.matmul(q.reshape(n, hk, g * l, d), k.transpose(2, 3)).reshape(n, hk, g, l, s)
    x = torch.exp(x / math.sqrt(d) - st["lse"].reshape(n, hk, g, l, 1))
    lim = st["kv_lens"][:, None]
    if c["causal"]:
        lim = lim - l + 1 + torch.arange(l, device=q.device)
    seen = torch.arange(s, device=q.device) < lim.expand(n, l)[:, :, None]
    return st["mass"] + (x * seen[:, None, None]).sum((2, 3))


def _plain_evict(st):
    c = st["case"]
    K, V, mass, pos = st["K"], st["V"], st["mass"], st["pos"]
    rows, hk, s, d = K.shape
    n, budget = c["n"], c["budget"]
    lens = st["kv_lens"].repeat(rows // n)[:, None, None]
    nxt = st["next_pos"].repeat(rows // n)[:, None, None]
    slot = torch.arange(s, device=K.device)
    inside = slot < lens
    held = (pos < c["sinks"]) | (pos >= nxt - c["recent"])
    key = torch.where(held, torch.full_like(mass, math.inf), mass)
    key = torch.where(inside, key, torch.full_like(mass, -math.inf))
    order = key.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, slot.expand_as(order))
    kept = (rank < budget) & inside
    hole, mover = ~kept & (slot < budget) & inside, kept & (slot >= budget)
    movers = torch.full((rows, hk, s + 1), 0, device=K.device, dtype=torch.int64)
    movers.scatter_(2, torch.where(mover, mover.long().cumsum(2) - 1, s), slot.expand_as(order))
    src = torch.where(hole, movers.gather(2, (hole.long().cumsum(2) - 1).clamp(min=0)), slot.expand_as(order))
    new = lens.clamp(max=budget)
    live = slot < new
    mass_out = torch.where(live, mass.gather(2, src), torch.zeros_like(mass))
    pos_out = torch.where(live, pos.gather(2, src), torch.full_like(pos, -1))
    src_out = torch.where(live, src, torch.full_like(src, -1))[:, :, :budget].to(torch.int32)
    K[:, :, :budget] = K.gather(2, src[:, :, :budget, None].expand(rows, hk, budget, d))
    V[:, :, :budget] = V.gather(2, src[:, :, :budget, None].expand(rows, hk, budget, d))
    return st["kv_lens"].clamp(max=budget), mass_out, pos_out, src_out, K, V


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    op, n = case["op"], case["n"]
    if op == "accept":
        l = case["l"]
        return {"bytes": (1 if case["shared"] else n) * l * 8 + n * l * 24 + n * 16, "flops": n * l}
    h, hk, d, e = case["h"], case["hk"], case["d"], _SIZE[case["dtype"]]
    lens = _lens(case)
    if op == "tree":
        l = case["l"]
        read = 2 * sum(lens) * hk * d * e + n * l * (h + 2 * hk) * d * e + n * l * l + n * 8
        return {"bytes": read + n * h * l * (d * e + 4), "flops": 4 * h * l * d * sum(x + l for x in lens)}
    if op == "append":
        rows = case["layers"] * sum(_counts(case))
        return {"bytes": rows * hk * (4 * d * e + 8) + n * 8 * (4 + case["l"]), "flops": 0}
    if op == "mass":
        l = case["l"]
        pairs = sum(x * l - (l * (l - 1) // 2 if case["causal"] else 0) for x in lens)
        return {"bytes": sum(lens) * hk * d * e + n * h * l * (d * e + 4) + 2 * n * hk * case["s"] * 4, "flops": 2 * h * d * pairs}
    rows, budget, s = case["layers"] * hk, case["budget"], case["s"]
    moved = 0
    for x in lens:
        if x > budget:                          # of the slots below the budget, the evicted share makes room
            recent = min(case["recent"], x - budget)
            free = x - case["sinks"] - case["recent"]
            moved += recent + (x - budget - recent) * (budget - case["sinks"] - case["recent"]) / max(1, free)
    return {"bytes": int(rows * (moved * d * e * 4 + sum(lens) * 8 + n * s * 8 + n * budget * 4)) + n * 24, "flops": 0}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "accept":
        return None                             # whole numbers
    st = prepare(case, seed)
    if op in ("append", "evict"):
        return _exact_moves(st)
    n, h, l, d = st["Q"].shape
    hk, g, lens = case["hk"], h // case["hk"], _lens(case)
    step = max(1, (1 << 27) // case["s"])       # query rows scored at a time
    if op == "mass":
        total = st["mass"].double()
        for b in range(n):
            for i in range(h):
                k = st["K"][b, i // g, :lens[b]].double()
                for a in range(0, l, step):
                    q = st["Q"][b, i, a:a + step].double()
                    w = torch.exp(q @ k.T * d ** -0.5 - st["lse"][b, i, a:a + step, None].double())
                    if case["causal"]:
                        w = w.tril(lens[b] - l + a)
                    total[b, i // g, :lens[b]] += w.sum(0)
        return total
    out = torch.zeros(n, h, l, d, device="cuda", dtype=torch.float64)
    lse = torch.full((n, h, l), -math.inf, device="cuda", dtype=torch.float64)
    for b in range(n):
        for i in range(h):
            q = st["Q"][b, i].double()
            near = (q @ st["Kd"][b, i // g].double().T).where(st["mask"][b], torch.tensor(-math.inf, device="cuda", dtype=torch.float64))
            score = torch.cat([q @ st["K"][b, i // g, :lens[b]].double().T, near], 1) * d ** -0.5
            value = torch.cat([st["V"][b, i // g, :lens[b]], st["Vd"][b, i // g]], 0).double()
            lse[b, i] = score.logsumexp(1)
            out[b, i] = (score - lse[b, i][:, None]).exp() @ value
    return out, lse


def _exact_moves(st):
    """Payloads are moved, not computed: row by row, from the definitions."""
    c, n, lens = st["case"], st["case"]["n"], _lens(st["case"])
    K, V, pos, mass = st["K"], st["V"], st["pos"], st["mass"]
    rows, hk, s, _ = K.shape
    if c["op"] == "append":
        counts, path, nxt = _counts(c), st["path"].tolist(), st["next_pos"].tolist()
        for r in range(rows):
            b = r % n
            at, take = slice(lens[b], lens[b] + counts[b]), path[b][:counts[b]]
            K[r, :, at], V[r, :, at] = st["Kd"][r][:, take], st["Vd"][r][:, take]
            mass[r, :, at] = 0.0
        return None, K.double(), V.double(), None, mass.double()
    budget = c["budget"]
    out = torch.zeros_like(mass, dtype=torch.float64)
    for r in range(rows):
        b = r % n
        new = min(lens[b], budget)
        out[r, :, :new] = mass[r, :, :new].double()
        if lens[b] <= budget:
            continue
        for i in range(hk):
            p, m = pos[r, i, :lens[b]], mass[r, i, :lens[b]]
            held = (p < c["sinks"]) | (p >= lens[b] - c["recent"])
            rest = torch.nonzero(~held)[:, 0]
            best = rest[m[rest].sort(dim=0, descending=True, stable=True).indices[:budget - int(held.sum())]]
            keep = held.clone()
            keep[best] = True
            free, come = torch.nonzero(~keep[:budget])[:, 0], budget + torch.nonzero(keep[budget:])[:, 0]
            K[r, i, free], V[r, i, free] = K[r, i, come], V[r, i, come]
            out[r, i, free] = m[come].double()
    return None, out, None, None, K.double(), V.double()
