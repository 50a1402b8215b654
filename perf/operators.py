"""What is timed of the operators on rows in groups: rows grouped by an index, matrix products over ragged groups with
their gradients, the weighted sum that joins a token's rows again, and low-rank adapters beside a shared projection.

A case is a dict of plain values.  prepare() makes what a program holds before the call, run() makes one pass: the plain
form in elementary torch operations, or, where `own` is set, the framework's calls.  exact() is the same in 64 bits."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "f64": 8}
DEVICE = "cuda:0"


# ------------------------------------------------------------------------------------------------------ the cases
def _case(name, op, **kw):
    c = {"name": name, "op": op, "dtype": "bf16", "tokens": 1, "fan": 1, "groups": 1, "k": 1, "n": 1, "rank": 0,
         "layout": "k", "dropped": 0.0}
    c.update(kw)
    return c


def listed():
    return [
        # one decoding step of a served batch: every sequence's token has chosen 8 of 128 experts; latency alone counts
        _case("group decode", "group", tokens=32, fan=8, groups=128),
        # the longest prefill or a training step: a million choices, some of them dropped by a capacity limit
        _case("group prefill", "group", tokens=131072, fan=8, groups=256, dropped=0.02),
        # the experts' first product in a decoding step: few rows for each expert, the weights are what is read
        _case("experts decode", "ragged", tokens=48, fan=4, groups=64, k=2048, n=1024),
        # the same in a long prefill: a thousand rows for each expert, bound by the matrix cores
        _case("experts prefill", "ragged", tokens=16384, fan=4, groups=64, k=2048, n=2048),
        # sizes that no tile divides and rows that start at any 2-byte address, weights with their columns contiguous
        _case("experts odd f16", "ragged", dtype="f16", tokens=1500, fan=2, groups=8, k=1001, n=777, layout="n", dropped=0.03),
        # a training step's gradients of the tokens and of every expert's weights
        _case("experts backward", "ragged_backward", tokens=8192, fan=4, groups=32, k=2048, n=1024, layout="n", dropped=0.01),
        # the blocks of a block-sparse contraction in double precision, rows already in order
        _case("blocks f64", "ragged", dtype="f64", tokens=24000, fan=1, groups=48, k=512, n=384, layout="n"),
        # the experts' results joined again, token by token, with the router's weights
        _case("combine prefill", "combine", tokens=16384, fan=4, groups=64, n=2048, dropped=0.02),
        # and its gradients, of the rows and of the router's weights
        _case("combine backward", "combine_backward", tokens=8192, fan=4, groups=32, n=2048, dropped=0.02),
        # a decoding step of 64 requests that use 32 fine-tuned adapters of one model, some of them none
        _case("adapters decode", "adapter", tokens=64, groups=32, k=4096, n=4096, rank=16, dropped=0.1),
        # prefill of a batch of requests with adapters
        _case("adapters prefill", "adapter", tokens=8192, groups=16, k=4096, n=4096, rank=32, dropped=0.1),
        # fine-tuning of several adapters at once on one frozen projection
        _case("adapters backward", "adapter_backward", tokens=4096, groups=8, k=4096, n=2048, rank=64),
    ]


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["group", "ragged", "ragged", "ragged_backward", "combine", "combine_backward", "adapter", "adapter",
                     "adapter_backward"])
    c = _case("", op)
    del c["name"]
    c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32", "f64"])
    c["layout"] = rng.choice(["k", "n"])
    c["dropped"] = rng.choice([0.0, 0.02, 0.1])
    top = max(_cost(x) for x in listed())
    if op == "group":
        c["dtype"] = "bf16"
        c["groups"] = _log(rng, 2, 512)
        c["fan"] = rng.randint(1, min(8, c["groups"]))
        c["tokens"] = _log(rng, 1, 131072)
        return c

    def width():  # half of them multiples of 64, as models have them, the others any number
        return 64 * _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 33, 4096)

    c["k"], c["n"] = (1 if op.startswith("combine") else width()), width()
    c["tokens"] = _log(rng, 1, 16384)
    if op.startswith("adapter"):
        c["groups"] = _log(rng, 1, 64)
        c["rank"] = rng.choice([4, 8, 16, 24, 32, 64, 7, 50])
    else:
        c["groups"] = _log(rng, 2, 128)
        c["fan"] = rng.randint(1, min(8, c["groups"]))
        while c["groups"] * c["k"] * c["n"] * SIZE[c["dtype"]] > 1 << 30:
            c["groups"] = max(2, c["groups"] // 2)
            c["fan"] = min(c["fan"], c["groups"])
            if c["groups"] == 2:
                break
    slow = {"bf16": 1, "f16": 1, "f32": 8, "f64": 16}[c["dtype"]]  # these types' rates are that much lower
    while c["tokens"] > 1 and _cost(c) * (slow if c["k"] > 1 else 1) > top:
        c["tokens"] = c["tokens"] * 2 // 3
    return c


def work(c):
    t, f, g, k, n, r, s = c["tokens"], c["fan"], c["groups"], c["k"], c["n"], c["rank"], SIZE[c["dtype"]]
    rows = t * f
    used = min(g, rows)  # no more groups than rows have rows in them
    if c["op"] == "group":  # the indices once (64 bits); offsets, order and positions once
        return {"bytes": 8 * rows + 8 * rows + 4 * (g + 1), "flops": 0}
    if c["op"] == "ragged":
        return {"bytes": s * (t * k + used * k * n + rows * n) + 4 * rows, "flops": 2 * rows * k * n}
    if c["op"] == "ragged_backward":  # tokens, weights, the gradient; the tokens' and all weights' gradients
        return {"bytes": s * (2 * t * k + used * k * n + g * k * n + rows * n) + 4 * rows, "flops": 4 * rows * k * n}
    if c["op"] == "combine":
        return {"bytes": s * (rows * n + t * n) + 8 * rows, "flops": 2 * rows * n}
    if c["op"] == "combine_backward":
        return {"bytes": s * (2 * rows * n + t * n) + 12 * rows, "flops": 3 * rows * n}
    low = s * min(g, t) * r * (k + n)
    if c["op"] == "adapter":
        return {"bytes": s * (t * k + k * n + t * n) + low, "flops": 2 * t * (k * n + r * (k + n))}
    return {"bytes": s * (2 * t * k + k * n + t * n) + 2 * low, "flops": 2 * t * (k * n + 3 * r * (k + n))}


# ------------------------------------------------------------------------------------------------------ the inputs
def _choices(c, rng):
    """int64 [tokens, fan]: what a router has chosen, some groups more often than others, each at most once for a token;
    -1 where a choice was dropped.  For adapters: one index a token, the same over a request's tokens."""
    t, f, g = c["tokens"], c["fan"], c["groups"]
    if c["op"].startswith("adapter"):
        if t <= 256:  # a decoding step: every token is another request's
            ids = torch.randint(0, g, (t,), generator=rng, device=DEVICE)
            gone = torch.rand(t, generator=rng, device=DEVICE) < c["dropped"]
            return torch.where(gone, -1, ids)[:, None]
        requests = min(t // 64, 2 * g)
        of = torch.randint(0, g, (requests,), generator=rng, device=DEVICE)
        of = torch.where(torch.rand(requests, generator=rng, device=DEVICE) < c["dropped"], -1, of)
        ends = torch.sort(torch.randint(0, t + 1, (requests - 1,), generator=rng, device=DEVICE)).values
        return of[torch.searchsorted(ends, torch.arange(t, device=DEVICE), right=True)][:, None]
    scores = torch.randn(t, g, generator=rng, device=DEVICE) + 0.3 * torch.randn(g, generator=rng, device=DEVICE)
    ids = torch.topk(scores, f, dim=1).indices
    gone = torch.rand(t, f, generator=rng, device=DEVICE) < c["dropped"]
    return torch.where(gone, -1, ids)


def _grouped(ids, g):
    """Offsets of the groups, the order that lists the rows group by group (rows of none at the end), and where each row
    has gone (-1 for those of none)."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < g), flat, g)
    sorted_key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(sorted_key, torch.arange(g + 1, device=key.device))
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel(), device=key.device)
    positions = torch.where(key < g, positions, -1)
    return offsets.to(torch.int32), order.to(torch.int32), positions.to(torch.int32)


def _weights(c, rows, columns, rng, scale):
    """[groups, rows, columns] with the layout's direction contiguous: "k" the rows, as a linear layer keeps them, "n" the columns."""
    dt = DTYPES[c["dtype"]]
    shape = (c["groups"], rows, columns) if c["layout"] == "n" else (c["groups"], columns, rows)
    w = torch.empty(shape, device=DEVICE, dtype=dt).normal_(0.0, scale, generator=rng)
    return w if c["layout"] == "n" else w.transpose(1, 2)


def prepare(case, seed):
    c = case
    rng = torch.Generator(device=DEVICE)
    rng.manual_seed(seed)
    dt, t, f, g, k, n, r = DTYPES[c["dtype"]], c["tokens"], c["fan"], c["groups"], c["k"], c["n"], c["rank"]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, device=DEVICE, dtype=dt).normal_(0.0, scale, generator=rng)

    ids = _choices(c, rng)
    s = {"case": c, "ids": ids}
    if c["op"] == "group":
        return s
    s["offsets"], s["order"], s["positions"] = _grouped(ids, g)
    if c["op"] in ("ragged", "ragged_backward"):
        s["x"], s["w"] = normal(t, k), _weights(c, k, n, rng, k ** -0.5)
        if c["op"] == "ragged_backward":
            s["dy"] = normal(t * f, n)
    elif c["op"] in ("combine", "combine_backward"):
        s["x"] = normal(t * f, n)
        wt = torch.float64 if dt == torch.float64 else torch.float32
        s["gates"] = torch.softmax(torch.randn(t, f, generator=rng, device=DEVICE, dtype=wt), dim=1)
        if c["op"] == "combine_backward":
            s["dy"] = normal(t, n)
    else:
        s["x"] = normal(t, k)
        s["w"] = _weights(dict(c, groups=1), k, n, rng, k ** -0.5)[0]
        s["a"], s["b"] = _weights(c, k, r, rng, k ** -0.5), _weights(c, r, n, rng, r ** -0.5)
        wt = torch.float64 if dt == torch.float64 else torch.float32
        s["scales"] = 0.25 + torch.rand(g, generator=rng, device=DEVICE, dtype=wt)
        if c["op"] == "adapter_backward":
            s["dy"] = normal(t, n)
    return s


# ------------------------------------------------------------------------------------------------------ the plain forms
def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _slots(s):
    """The place of each row in order in a [groups, longest group] array, the rows of no group left out."""
    o = s["offsets"].long()
    longest = int((o[1:] - o[:-1]).max())
    p = torch.arange(int(o[-1]), device=o.device)
    group = torch.searchsorted(o[1:], p, right=True)
    return group, p - o[group], longest


def _padded(x, s, at):
    group, place, longest = at
    out = torch.zeros(s["case"]["groups"], longest, x.shape[1], dtype=x.dtype, device=x.device)
    out[group, place] = x[:group.numel()]
    return out


def _plain_ragged(s):
    x, w, at = _wide(s["x"]), _wide(s["w"]), _slots(s)
    source = s["order"].long() // s["case"]["fan"]
    y = torch.zeros(source.numel(), w.shape[2], dtype=x.dtype, device=x.device)
    y[:at[0].numel()] = torch.matmul(_padded(x[source], s, at), w)[at[0], at[1]]
    return y.to(s["x"].dtype)


def _plain_ragged_backward(s):
    x, w, dy, at = _wide(s["x"]), _wide(s["w"]), _wide(s["dy"]), _slots(s)
    source = s["order"].long() // s["case"]["fan"]
    xp, dyp = _padded(x[source], s, at), _padded(dy, s, at)
    dw = torch.matmul(xp.transpose(1, 2), dyp)
    rows = torch.zeros(source.numel(), x.shape[1], dtype=x.dtype, device=x.device)
    rows[s["order"].long()[:at[0].numel()]] = torch.matmul(dyp, w.transpose(1, 2))[at[0], at[1]]
    dx = rows.view(x.shape[0], s["case"]["fan"], -1).sum(1)
    return dx.to(s["x"].dtype), dw.to(s["w"].dtype)


def _plain_combine(s):
    place = s["positions"].long().view(s["gates"].shape)
    gates = torch.where(place >= 0, s["gates"], 0.0)
    return torch.sum(gates[:, :, None] * _wide(s["x"])[place.clamp(min=0)], dim=1).to(s["x"].dtype)


def _plain_combine_backward(s):
    place = s["positions"].long().view(s["gates"].shape)
    dy = _wide(s["dy"])
    dgates = torch.where(place >= 0, torch.sum(_wide(s["x"])[place.clamp(min=0)] * dy[:, None, :], dim=2), 0.0)
    order = s["order"].long()
    gate = torch.where(s["positions"] >= 0, s["gates"].reshape(-1), 0.0)[order]
    dx = gate[:, None] * dy[order // s["case"]["fan"]]
    return dx.to(s["x"].dtype), dgates


def _plain_low_rank(x, a, b, scales, s, at):
    """Each row's scale * (x a) b in the rows' own order, and the middle (x a) and its rows padded by group."""
    rows = s["order"].long()[:at[0].numel()]
    xp = _padded(x[rows], s, at)
    middle = torch.matmul(xp, a)
    out = torch.zeros(x.shape[0], b.shape[2], dtype=x.dtype, device=x.device)
    out[rows] = (torch.matmul(middle, b) * scales[:, None, None])[at[0], at[1]]
    return out, xp, middle


def _plain_adapter(s):
    x, at = _wide(s["x"]), _slots(s)
    return (x @ _wide(s["w"]) + _plain_low_rank(x, _wide(s["a"]), _wide(s["b"]), s["scales"], s, at)[0]).to(s["x"].dtype)


def _plain_adapter_backward(s):
    x, dy, a, b, at = _wide(s["x"]), _wide(s["dy"]), _wide(s["a"]), _wide(s["b"]), _slots(s)
    low, dyp, back = _plain_low_rank(dy, b.transpose(1, 2), a.transpose(1, 2), s["scales"], s, at)
    xp = _padded(x[s["order"].long()[:at[0].numel()]], s, at)
    scale = s["scales"][:, None, None]
    da = scale * torch.matmul(xp.transpose(1, 2), back)
    db = scale * torch.matmul(torch.matmul(xp, a).transpose(1, 2), dyp)
    dx = dy @ _wide(s["w"]).t() + low
    return dx.to(s["x"].dtype), da.to(s["a"].dtype), db.to(s["b"].dtype)


# ------------------------------------------------------------------------------------------------------ one pass
def _own(s):
    import tenferro_rs_amd as tf
    c = s["case"]
    if c["op"] == "group":
        g = tf.RowGroups.from_ids(s["ids"], c["groups"])
        return g.offsets, g.order, g.positions
    groups = tf.RowGroups(s["offsets"], s["order"], s["positions"], fan=c["fan"])
    if c["op"] == "ragged":
        return tf.ragged_gemm(s["x"], s["w"], groups, gather=True)
    if c["op"] == "ragged_backward":
        return tf.ragged_gemm_backward(s["x"], s["w"], s["dy"], groups, gather=True)
    if c["op"] == "combine":
        return tf.combine_rows(s["x"], groups, s["gates"])
    if c["op"] == "combine_backward":
        return tf.combine_rows_backward(s["x"], s["gates"], s["dy"], groups)
    if c["op"] == "adapter":
        return tf.adapter_gemm(s["x"], s["w"], s["a"], s["b"], groups, s["scales"])
    return tf.adapter_gemm_backward(s["x"], s["w"], s["a"], s["b"], s["dy"], groups, s["scales"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "group":
        return _grouped(state["ids"], state["case"]["groups"])
    return {"ragged": _plain_ragged, "ragged_backward": _plain_ragged_backward, "combine": _plain_combine,
            "combine_backward": _plain_combine_backward, "adapter": _plain_adapter,
            "adapter_backward": _plain_adapter_backward}[op](state)


# ------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    g, f = c["groups"], c["fan"]
    ids = s["ids"].reshape(-1).cpu().numpy()
    members = [np.nonzero(ids == i)[0] for i in range(g)]
    rest = np.nonzero((ids < 0) | (ids >= g))[0]
    listing = np.concatenate(members + [rest])
    if c["op"] == "group":
        offsets = np.cumsum([0] + [len(m) for m in members])
        positions = np.full(len(ids), -1)
        positions[listing[:offsets[-1]]] = np.arange(offsets[-1])
        return tuple(torch.from_numpy(v.astype(np.int32)) for v in (offsets, listing, positions))
    on = [torch.from_numpy(m).to(DEVICE) for m in members]  # the flat rows of each group
    start = np.cumsum([0] + [len(m) for m in members])
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=DEVICE)  # noqa: E731
    if c["op"] == "ragged":
        y = zeros(len(ids), c["n"])
        for i, m in enumerate(on):
            y[start[i]:start[i + 1]] = d["x"][m // f] @ d["w"][i]
        return y
    if c["op"] == "ragged_backward":
        dx, dw = zeros(c["tokens"], c["k"]), zeros(g, c["k"], c["n"])
        for i, m in enumerate(on):
            part = d["dy"][start[i]:start[i + 1]]
            dx.index_add_(0, m // f, part @ d["w"][i].t())
            dw[i] = d["x"][m // f].t() @ part
        return dx, dw
    if c["op"] == "combine":
        y = zeros(c["tokens"], c["n"])
        for i, m in enumerate(on):
            y.index_add_(0, m // f, d["gates"].reshape(-1)[m][:, None] * d["x"][start[i]:start[i + 1]])
        return y
    if c["op"] == "combine_backward":
        dx, dg = zeros(len(ids), c["n"]), zeros(c["tokens"] * f)
        for i, m in enumerate(on):
            dx[start[i]:start[i + 1]] = d["gates"].reshape(-1)[m][:, None] * d["dy"][m // f]
            dg[m] = (d["x"][start[i]:start[i + 1]] * d["dy"][m // f]).sum(1)
        return dx, dg.view(c["tokens"], f)
    if c["op"] == "adapter":
        y = d["x"] @ d["w"]
        for i, m in enumerate(on):
            y[m] += d["scales"][i] * (d["x"][m] @ d["a"][i] @ d["b"][i])
        return y
    dx, da, db = d["dy"] @ d["w"].t(), zeros(g, c["k"], c["rank"]), zeros(g, c["rank"], c["n"])
    for i, m in enumerate(on):
        x, dy = d["x"][m], d["dy"][m]
        dx[m] += d["scales"][i] * (dy @ d["b"][i].t() @ d["a"][i].t())
        da[i] = d["scales"][i] * (x.t() @ (dy @ d["b"][i].t()))
        db[i] = d["scales"][i] * ((x @ d["a"][i]).t() @ dy)
    return dx, da, db
