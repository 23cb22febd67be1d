"""Performance cases of the operators on device tensors: lookup in a table and its gradient, rows to their clusters and back,
products in 8 bits.

A case is a dict of plain values.  `listed()` gives the fixed ones, `draw()` further ones of the same ranges; `prepare()` makes
the inputs of a case on the GPU from a seed, `run()` makes one pass: in elementary torch operations, or, where `own` is true,
through superkmeans_b200.ops.  `exact()` is what a pass returns, from the definition in 64 bits.

The definitions:
  lookup     out[i] = scale * row_scales[i] * table[ids[i]]; an id outside the table gives a row of zeros
  its gradient  grad_table[c] = sum over ids[i] = c of scale * row_scales[i] * grad[i]; grad_row_scales[i] = scale * <grad[i], table[ids[i]]>
  route      the (row, choice) pairs in the order of their cluster, ties in their own order (order, its inverse `position`, and where
             each cluster begins; pairs without a cluster come last); the rows in that order; and from other rows in that order
             out[i] = sum over j of weights[i][j] * y[position[i][j]]
  its gradient  of y, weights and the rows
  product    out[i][c] = x_scale[i] * w_scale[c] * sum over j of q[i][j] * w[c][j], for rows in clusters with the w of the row's cluster;
             q[i] = rint(x[i] * (127 / largest |x[i]|)), x_scale[i] = largest / 127 where the rows are not in 8 bits already
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
SKEW = 0.9   # share of cluster j of a collection: (j + 5) ** -SKEW, as cluster sizes of embeddings fall off


def listed():
    return [
        # ---- lookup
        # the vectors of one batch of tokens from a codebook of 1000: nothing but latency
        dict(name="lookup_batch", call="lookup", n=256, k=1_000, d=768, dtype="fp32", scale=1.0, row_scales=False, lost=0.0),
        # a collection decoded from its assignments, unit centroids times each row's norm
        dict(name="lookup_collection", call="lookup", n=1_000_000, k=65_536, d=768, dtype="bf16", scale=1.0, row_scales=True, lost=0.0),
        # a codebook trained with a model on small batches, odd width, norms trained too, a tenth of the places padding
        dict(name="lookup_grad_odd", call="lookup_grad", n=2_001, k=300, d=130, dtype="fp16", scale=11.4, row_scales=True, lost=0.1),
        # the gradient of a large table after a large batch
        dict(name="lookup_grad_large", call="lookup_grad", n=500_000, k=16_384, d=1_024, dtype="bf16", scale=32.0, row_scales=False, lost=0.0),
        # ---- rows to their clusters and back
        # a step of a server: a few rows, two clusters each
        dict(name="route_step", call="route", n=64, m=2, k=16, d=1_024, dtype="bf16", lost=0.0),
        # a training batch, some choices dropped
        dict(name="route_batch", call="route", n=131_072, m=2, k=256, d=1_024, dtype="bf16", lost=0.02),
        # many clusters, four each, odd counts, fp32
        dict(name="route_many", call="route", n=30_001, m=4, k=10_000, d=384, dtype="fp32", lost=0.0),
        # the backward pass of a training batch
        dict(name="route_grad_batch", call="route_grad", n=131_072, m=2, k=256, d=768, dtype="bf16", lost=0.02),
        # ---- products in 8 bits
        # one query against the centroids of the two-level configuration's leaves: the weights' bytes and latency
        dict(name="product_query", call="product", n=1, m=16_384, d=768, groups=0, dtype="fp32", given=False, pitched=True),
        # a batch of rows of odd width
        dict(name="product_odd", call="product", n=777, m=1_001, d=130, groups=0, dtype="fp16", given=False, pitched=False),
        # stored rows against the headline configuration's centroids
        dict(name="product_scores", call="product", n=32_768, m=10_000, d=1_024, groups=0, dtype="bf16", given=True, pitched=True),
        # rows of 256 coarse clusters times a matrix of each cluster's own
        dict(name="product_by_cluster", call="product", n=65_536, m=768, d=768, groups=256, dtype="bf16", given=False, pitched=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def _width(rng, lo, hi):
    """A row width: usually a multiple of 8, one in four as it falls."""
    d = _log_int(rng, lo, hi)
    return d if rng.random() < 0.25 else max(8, d // 8 * 8)


def draw(rng):
    call = rng.choice(["lookup", "lookup_grad", "route", "route_grad", "product", "product"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    d = _width(rng, 16, 1_536)
    if call in ("lookup", "lookup_grad"):
        k = _log_int(rng, 16, 65_536)
        most = min(1_000_000, int((1.2e9 if call == "lookup" else 9e8) / (d * SIZES[dtype])))
        return dict(call=call, n=_log_int(rng, 1, most), k=k, d=d, dtype=dtype, scale=rng.choice([1.0, round(math.sqrt(d), 3)]), row_scales=rng.random() < 0.5, lost=rng.choice([0.0, 0.0, 0.1]))
    if call in ("route", "route_grad"):
        m, k = rng.choice([1, 2, 2, 4, 8]), _log_int(rng, 8, 16_384)
        most = min(200_000, int((4e8 if call == "route" else 3e8) / (m * d * SIZES[dtype])))
        return dict(call=call, n=_log_int(rng, 1, most), m=m, k=k, d=d, dtype=dtype, lost=rng.choice([0.0, 0.02, 0.3]))
    groups = 0 if rng.random() < 0.6 else _log_int(rng, 2, 512)
    m = _log_int(rng, 16, 10_000 if groups == 0 else min(2_048, int(1.5e8 / (groups * d))))
    most = min(65_536, int(3e8 / m), int(2e8 / d))
    return dict(call=call, n=_log_int(rng, 1, most), m=m, d=d, groups=groups, dtype=dtype, given=rng.random() < 0.3, pitched=rng.random() < 0.7)


# ---- inputs -------------------------------------------------------------------------------------------------------------------


def _shares(k):
    return (torch.arange(k, dtype=torch.float64) + 5.0) ** -SKEW


def _ids(g, n, k):
    """Clusters of n rows; their sizes fall off, and the large ones are spread over the numbers."""
    cumulative = torch.cumsum(_shares(k), 0).cuda()
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * cumulative[-1]
    ranked = torch.searchsorted(cumulative, u).clamp_(max=k - 1)
    return torch.randperm(k, generator=g, device="cuda")[ranked].to(torch.int32)


def _choices(g, n, m, k, lost):
    """m clusters for each row, of a router that is roughly balanced; some of them given up (-1)."""
    lean = torch.randn(min(k, 4096), generator=g, device="cuda") * 0.5
    at = torch.multinomial(torch.softmax(lean, 0), n * m, replacement=True, generator=g)
    at = (at + torch.randint(0, -(-k // lean.numel()), (n * m,), generator=g, device="cuda") * lean.numel()) % k
    ids = at.to(torch.int32)
    if lost:
        ids[torch.rand(n * m, generator=g, device="cuda") < lost] = -1
    return ids.reshape(n, m)


def _weights(g, n, m):
    return torch.softmax(torch.randn(n, m, generator=g, device="cuda"), 1)


def _rows(g, n, d, dtype, unit=False):
    """Rows whose lengths differ, as activations' and gradients' do; with `unit` of length one."""
    x = torch.randn(n, d, generator=g, device="cuda")
    if unit:
        return (x / x.square().sum(1, keepdim=True).sqrt()).to(TYPES[dtype])
    return (x * torch.exp(0.5 * torch.randn(n, 1, generator=g, device="cuda"))).to(TYPES[dtype])


def _bytes_of(x):
    """Rows in 8 bits with a scale each, as they are stored."""
    largest = x.abs().amax(-1)
    return torch.round(x * (127.0 / largest)[..., None]).to(torch.int8), largest / 127.0


def _pitched(q, pitched):
    """The same rows, each beginning on 16 bytes if `pitched`."""
    if not pitched:
        return q.contiguous()
    d = q.shape[-1]
    room = torch.zeros(*q.shape[:-1], -(-d // 16) * 16, dtype=torch.int8, device=q.device)
    room[..., :d] = q
    return room[..., :d]


def _sorted_pairs(ids, k):
    """(order, position, offsets) of a route, for the state of its backward pass."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < k), flat, k)
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.searchsorted(key[order], torch.arange(k + 1, device=order.device))
    return order.to(torch.int32), position.reshape(ids.shape).to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    c = dict(case)
    n, d = c["n"], c["d"]
    if c["call"] in ("lookup", "lookup_grad"):
        c["ids"] = _ids(g, n, c["k"])
        if c["lost"]:
            c["ids"][torch.rand(n, generator=g, device="cuda") < c["lost"]] = -1
        c["table"] = _rows(g, c["k"], d, c["dtype"], unit=c["row_scales"])
        c["scales"] = torch.exp(0.3 * torch.randn(n, generator=g, device="cuda")) if c["row_scales"] else None
        if c["call"] == "lookup_grad":
            c["grad"] = _rows(g, n, d, c["dtype"])
    elif c["call"] in ("route", "route_grad"):
        m = c["m"]
        c["ids"] = _choices(g, n, m, c["k"], c["lost"])
        c["weights"] = _weights(g, n, m)
        c["y"] = _rows(g, n * m, d, c["dtype"])
        if c["call"] == "route":
            c["x"] = _rows(g, n, d, c["dtype"])
        else:
            c["groups"] = _sorted_pairs(c["ids"], c["k"])
            c["grad"] = _rows(g, n, d, c["dtype"])
            c["grad_rows"] = _rows(g, n * m, d, c["dtype"])
    else:
        e = max(1, c["groups"])
        w, c["w_scales"] = _bytes_of(_rows(g, e * c["m"], d, "fp32").reshape(e, c["m"], d))
        w = _pitched(w, c["pitched"])
        c["w"], c["w_scales"] = (w, c["w_scales"]) if c["groups"] else (w[0], c["w_scales"][0])
        c["x"] = _rows(g, n, d, c["dtype"])
        if c["given"]:
            q, c["x_scales"] = _bytes_of(c["x"].float())
            c["x"] = _pitched(q, c["pitched"])
        c["offsets"] = None
        if c["groups"]:
            sizes = torch.bincount(torch.sort(_choices(g, n, 1, e, 0.0).reshape(-1)).values, minlength=e)
            c["offsets"] = torch.cat([sizes.new_zeros(1), torch.cumsum(sizes, 0)]).to(torch.int32)
            c["most"] = int(sizes.max())   # (the host made the plan)
    return c


# ---- one pass -----------------------------------------------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from superkmeans_b200 import ops

    if s["call"] == "lookup":
        return ops.lookup(s["table"], s["ids"], s["scale"], s["scales"])
    if s["call"] == "lookup_grad":
        grad_table = ops.lookup_grad(s["grad"], s["ids"], s["k"], s["scale"], s["scales"])
        if s["scales"] is None:
            return grad_table
        return grad_table, ops.lookup_scale_grad(s["grad"], s["table"], s["ids"], s["scale"])
    if s["call"] == "route":
        groups = ops.group_rows(s["ids"], s["k"])
        return *groups, ops.to_clusters(s["x"], groups), ops.from_clusters(s["y"], groups, s["weights"])
    if s["call"] == "route_grad":
        groups = ops.RowGroups(*s["groups"])
        return *ops.from_clusters_grad(s["grad"], s["y"], groups, s["weights"]), ops.to_clusters_grad(s["grad_rows"], groups)
    q, scales = (s["x"], s["x_scales"]) if s["given"] else ops.quantize_rows(s["x"])
    return ops.product_8bit(q, scales, s["w"], s["w_scales"], s["offsets"], dtype=TYPES[s["dtype"]])


def _run_plain(s):
    if s["call"] in ("lookup", "lookup_grad"):
        return _plain_lookup(s)
    if s["call"] == "route":
        return _plain_route(s)
    if s["call"] == "route_grad":
        return _plain_route_grad(s)
    return _plain_product(s)


def _plain_lookup(s):
    ids, k = s["ids"].long(), s["k"]
    valid = (ids >= 0) & (ids < k)
    factor = torch.full((s["n"], 1), s["scale"], device=ids.device)
    if s["scales"] is not None:
        factor = factor * s["scales"][:, None]
    if s["call"] == "lookup":
        rows = s["table"].float()[torch.where(valid, ids, 0)] * factor
        return torch.where(valid[:, None], rows, 0.0).to(s["table"].dtype)
    # (sums over many rows: in 64 bits)
    sums = torch.zeros(k + 1, s["d"], dtype=torch.float64, device=ids.device)
    sums.index_add_(0, torch.where(valid, ids, k), s["grad"].double() * factor)
    grad_table = sums[:k].to(s["grad"].dtype)
    if s["scales"] is None:
        return grad_table
    dots = (s["grad"].float() * s["table"].float()[torch.where(valid, ids, 0)]).sum(1) * s["scale"]
    return grad_table, torch.where(valid, dots, 0.0)


def _plain_route(s):
    order, position, offsets = _sorted_pairs(s["ids"], s["k"])
    held = offsets[-1]
    slot = torch.arange(order.numel(), device=order.device)
    rows = torch.where((slot < held)[:, None], s["x"][order // s["m"]], 0.0)
    back = torch.where((position < held)[..., None], s["y"].float()[position.long()], 0.0)
    return order, position, offsets, rows, (back * s["weights"][..., None]).sum(1).to(s["y"].dtype)


def _plain_route_grad(s):
    order, position, offsets = s["groups"]
    held, m, kind = offsets[-1], s["m"], s["y"].dtype
    slot = torch.arange(order.numel(), device=order.device)
    grad_y = s["grad"].float()[order // m] * s["weights"].reshape(-1)[order.long()][:, None]
    grad_y = torch.where((slot < held)[:, None], grad_y, 0.0).to(kind)
    there = (position < held)[..., None]
    at = position.long()
    grad_weights = (torch.where(there, s["y"].float()[at], 0.0) * s["grad"].float()[:, None, :]).sum(2)
    grad_x = torch.where(there, s["grad_rows"].float()[at], 0.0).sum(1).to(kind)
    return grad_y, grad_weights, grad_x


def _plain_product(s):
    kind = TYPES[s["dtype"]]
    if s["given"]:
        q, scales = s["x"].float(), s["x_scales"]
    else:
        x = s["x"].float()
        largest = x.abs().amax(1)
        q, scales = torch.round(x * (127.0 / largest)[:, None]), largest / 127.0
    if not s["groups"]:
        return (q @ s["w"].float().T * scales[:, None] * s["w_scales"]).to(kind)
    # the rows of each cluster in a box of their own, as many rows as the largest cluster has
    row = torch.arange(s["n"], device=q.device)
    group = torch.searchsorted(s["offsets"][1:].contiguous(), row.to(torch.int32), right=True)
    place = group * s["most"] + (row - s["offsets"][group])
    boxes = torch.zeros(s["groups"] * s["most"], s["d"], device=q.device)
    boxes[place] = q
    sums = torch.bmm(boxes.reshape(s["groups"], s["most"], s["d"]), s["w"].float().transpose(1, 2))
    return (sums.reshape(-1, s["m"])[place] * scales[:, None] * s["w_scales"][group]).to(kind)


# ---- what a pass has to do ------------------------------------------------------------------------------------------------------


def _touched(n, k):
    p = _shares(k) / _shares(k).sum()
    return float((1.0 - torch.exp(n * torch.log1p(-p))).sum()) if k > 1 else 1.0


def work(case):
    c, n, d = case, case["n"], case["d"]
    t = SIZES[c["dtype"]]
    if c["call"] == "lookup":
        rows = _touched(n, c["k"])
        return {"bytes": n * (4 + (4 if c["row_scales"] else 0)) + (rows + n) * d * t, "flops": n * d}
    if c["call"] == "lookup_grad":
        scaled = n * 8 + _touched(n, c["k"]) * d * t if c["row_scales"] else 0
        return {"bytes": n * 4 + (n + c["k"]) * d * t + scaled, "flops": n * d * (4 if c["row_scales"] else 2)}
    if c["call"] == "route":
        pairs = n * c["m"]
        return {"bytes": pairs * (4 + 8 + 4) + c["k"] * 4 + (2 * n + 2 * pairs) * d * t, "flops": 2 * pairs * d}
    if c["call"] == "route_grad":
        pairs = n * c["m"]
        return {"bytes": pairs * 12 + (2 * n + 3 * pairs) * d * t, "flops": 4 * pairs * d}
    e = max(1, c["groups"])
    return {"bytes": n * d * (1 if c["given"] else t) + 4 * n + e * c["m"] * (d + 4) + n * c["m"] * t, "flops": 2 * n * c["m"] * d}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if s["call"] in ("lookup", "lookup_grad"):
        return _exact_lookup(s)
    if s["call"] in ("route", "route_grad"):
        return _exact_route(s)
    return _exact_product(s)


def _exact_lookup(s):
    n, k, d = s["n"], s["k"], s["d"]
    ids = s["ids"].long()
    there = torch.nonzero((ids >= 0) & (ids < k)).reshape(-1)
    factor = torch.full((n,), float(s["scale"]), dtype=torch.float64, device="cuda")
    if s["scales"] is not None:
        factor *= s["scales"].double()
    if s["call"] == "lookup":
        out = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        for piece in there.split(100_000):
            out[piece] = torch.einsum("i,ij->ij", factor[piece], s["table"].double().index_select(0, ids[piece]))
        return out
    # sums of sorted rows as differences of running sums, a column block at a time
    ids, grad = ids[there], s["grad"][there].double() * factor[there, None]
    by = torch.sort(ids).indices
    ends = torch.bincount(ids, minlength=k).cumsum(0)
    grad_table = torch.empty(k, d, dtype=torch.float64, device="cuda")
    for c0 in range(0, d, 128):
        running = torch.cat([grad.new_zeros(1, min(128, d - c0)), grad[by, c0:c0 + 128].cumsum(0)])
        at = running[ends]
        grad_table[:, c0:c0 + 128] = torch.diff(at, dim=0, prepend=torch.zeros_like(at[:1]))
    if s["scales"] is None:
        return grad_table
    dots = torch.zeros(n, dtype=torch.float64, device="cuda")
    for piece in there.split(100_000):
        dots[piece] = torch.einsum("ij,ij->i", s["grad"][piece].double(), s["table"].double()[s["ids"][piece].long()]) * float(s["scale"])
    return grad_table, dots


def _exact_route(s):
    n, m, k, d = s["n"], s["m"], s["k"], s["d"]
    flat = [c if 0 <= c < k else k for c in s["ids"].reshape(-1).tolist()]
    order = sorted(range(n * m), key=flat.__getitem__)
    held = sum(c < k for c in flat)
    order = torch.tensor(order, device="cuda")
    position = torch.zeros(n * m, dtype=torch.int64, device="cuda").scatter_(0, order, torch.arange(n * m, device="cuda"))
    live = order[:held]   # pairs that have a cluster, in their order
    w = s["weights"].double().reshape(-1)
    if s["call"] == "route":
        rows = torch.zeros(n * m, d, dtype=torch.float64, device="cuda")
        rows[:held] = s["x"].double().index_select(0, live // m)
        out = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        for j in range(m):
            mine = position.reshape(n, m)[:, j]
            i = torch.nonzero(mine < held).reshape(-1)
            out[i] += s["y"].double()[mine[i]] * w.reshape(n, m)[i, j, None]
        return None, None, None, rows, out
    grad, y, up = s["grad"].double(), s["y"].double(), s["grad_rows"].double()
    grad_y = torch.zeros(n * m, d, dtype=torch.float64, device="cuda")
    grad_y[:held] = torch.einsum("i,ij->ij", w[live], grad[live // m])
    grad_w = torch.zeros(n * m, dtype=torch.float64, device="cuda")
    grad_w[live] = torch.einsum("ij,ij->i", y[:held], grad[live // m])
    grad_x = torch.zeros(n, d, dtype=torch.float64, device="cuda")
    grad_x.index_add_(0, live // m, up[:held])
    return grad_y, grad_w.reshape(n, m), grad_x


def _exact_product(s):
    x = s["x"].double()
    if s["given"]:
        q, scales = x, s["x_scales"].double()
    else:
        most = x.abs().max(1).values
        q, scales = torch.round(x / most[:, None] * 127.0), most / 127.0
    w, ws = s["w"].double(), s["w_scales"].double()
    if not s["groups"]:
        return torch.einsum("ij,cj->ic", q * scales[:, None], w * ws[:, None])
    out = torch.empty(s["n"], s["m"], dtype=torch.float64, device="cuda")
    ends = s["offsets"].tolist()
    for e in range(s["groups"]):
        a, b = ends[e], ends[e + 1]
        out[a:b] = torch.einsum("ij,cj->ic", q[a:b] * scales[a:b, None], w[e] * ws[e][:, None])
    return out
