"""The routed products of a mixture: what is measured of them, and their plain forms.

Four operators, each with the call a user makes of ``gmmxx_b200`` (``own``)
and its plain form in elementary torch operations:

* route       -- rows sorted by the component they are assigned to
* forward     -- each row times its component's matrix (plus bias), from labels
* step        -- the same with the gradients of rows, matrices and biases
* orthogonal  -- Newton-Schulz orthogonalisation of a stack of matrices
"""

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # two experts for each of 32 rows of a serving batch: nothing but latency
        dict(name="route_serving", op="route", rows=32, top=2, groups=16, index="int64", dropped=0.0),
        # a batch of 8191 rows, two experts each, one row in fifty left unassigned
        dict(name="route_batch", op="route", rows=8191, top=2, groups=64, index="int32", dropped=0.02),
        # 4.2M rows over the 8192 components of a large spherical mixture
        dict(name="route_cells", op="route", rows=1 << 22, top=1, groups=8192, index="int64", dropped=0.0),
        # the serving batch's products: bound by reading the chosen experts' weights
        dict(name="forward_serving", op="forward", rows=32, top=2, groups=16, n_in=2048, n_out=1024, dtype="bf16",
             bias=True, dropped=0.0),
        # a whole batch, two experts per row, wide experts: bound by the products
        dict(name="forward_batch", op="forward", rows=8191, top=2, groups=16, n_in=2048, n_out=4096, dtype="bf16",
             bias=False, dropped=0.0),
        # each component's own 64 x 64 map applied to its rows (fp32 rows as the tied fits take them)
        dict(name="forward_cells", op="forward", rows=262144, top=1, groups=256, n_in=64, n_out=64, dtype="fp32",
             bias=True, dropped=0.0),
        # one training step of the wide experts
        dict(name="step_batch", op="step", rows=8192, top=2, groups=16, n_in=2048, n_out=4096, dtype="bf16",
             bias=False, dropped=0.0),
        # a training step of per-component maps of 128 dimensions, as many rows as fit a fit's chunk
        dict(name="step_cells", op="step", rows=500009, top=1, groups=512, n_in=128, n_out=128, dtype="bf16",
             bias=True, dropped=0.01),
        # odd widths, an odd number of components, fp16
        dict(name="step_odd", op="step", rows=5003, top=1, groups=37, n_in=1001, n_out=1531, dtype="fp16",
             bias=True, dropped=0.0),
        # a rotation for each of 512 components of 64 dimensions
        dict(name="orthogonal_components", op="orthogonal", batch=512, m=64, n=64, steps=5, dtype="fp32"),
        # the update of one layer's sixteen experts
        dict(name="orthogonal_experts", op="orthogonal", batch=16, m=2048, n=1024, steps=5, dtype="bf16"),
        # the update of one odd-sized wide matrix
        dict(name="orthogonal_matrix", op="orthogonal", batch=1, m=1000, n=4095, steps=5, dtype="fp32"),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "forward", "step", "orthogonal"])
    if op == "route":
        top = rng.choice([1, 1, 2, 4, 8])
        return dict(op=op, rows=_spread(rng, 16, (1 << 22) // top), top=top, groups=_spread(rng, 2, 8192),
                    index=rng.choice(["int64", "int32"]), dropped=rng.choice([0.0, 0.0, 0.03]))
    if op == "orthogonal":
        m, n = _spread(rng, 16, 2048), _spread(rng, 16, 2048)
        cost = min(m, n) ** 2 * max(m, n)
        most = max(1, min(512, (1 << 34) // cost))
        return dict(op=op, batch=_spread(rng, 1, most), m=m, n=n, steps=rng.choice([3, 5, 5, 6]),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]))
    top = rng.choice([1, 1, 2, 4])
    groups = _spread(rng, 3, 256)
    n_in, n_out = _spread(rng, 32, 4096), _spread(rng, 32, 4096)
    if rng.random() < 0.5:  # half of them in steps of 32 as models have them, the others as they fall
        n_in, n_out = (n_in + 31) // 32 * 32, (n_out + 31) // 32 * 32
    groups = max(1, min(groups, (1 << 27) // (n_in * n_out)))
    rows = _spread(rng, 8, max(16, min(262144, (1 << 36) // (n_in * n_out * top))))
    return dict(op=op, rows=rows, top=top, groups=groups, n_in=n_in, n_out=n_out,
                dtype=rng.choice(["bf16", "fp16", "fp32"]), bias=rng.random() < 0.5,
                dropped=rng.choice([0.0, 0.0, 0.03]))


def _labels(case, gen):
    """Labels as an uneven mixture gives them: some components take several
    times the rows of others; -1 where a row's choice was dropped."""
    k, shape = case["groups"], (case["rows"], case["top"])
    share = torch.exp(0.5 * torch.randn(k, generator=gen, device="cuda"))
    edges = torch.cumsum(share / share.sum(), 0)
    u = torch.rand(shape, generator=gen, device="cuda")
    labels = torch.searchsorted(edges, u).clamp_max(k - 1)
    lost = torch.rand(shape, generator=gen, device="cuda") < case["dropped"]
    labels = torch.where(lost, torch.full_like(labels, -1), labels)
    return labels.squeeze(1) if case["top"] == 1 else labels


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    state = dict(case)
    if case["op"] == "orthogonal":
        # an update as training gives it: directions of very different weight
        m, n, b = case["m"], case["n"], case["batch"]
        scale = torch.exp(normal(b, m, 1)) * 0.01
        state["update"] = (normal(b, m, n) * scale).to(DTYPES[case["dtype"]])
        return state
    labels = _labels(case, gen)
    counts = torch.bincount(labels.reshape(-1).clamp_min(0), minlength=case["groups"])
    state["most"] = int(counts.max())  # rows of the fullest group (the dropped counted to the first)
    if case["op"] == "route":
        state["labels"] = labels.to(torch.int32 if case["index"] == "int32" else torch.int64)
        return state
    state["labels"] = labels
    dt, n_in, n_out, k = DTYPES[case["dtype"]], case["n_in"], case["n_out"], case["groups"]
    state["x"] = normal(case["rows"], n_in).to(dt)
    state["weight"] = (normal(k, n_in, n_out) / n_in**0.5).to(dt)
    state["bias"] = normal(k, n_out).to(dt) if case["bias"] else None
    if case["op"] == "step":
        state["grad"] = normal(*labels.shape, n_out).to(dt)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _sorted_rows(labels, k):
    flat = labels.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < k), flat, torch.full_like(flat, k))
    order = torch.argsort(key, stable=True)
    ends = torch.cumsum(torch.bincount(key, minlength=k + 1), 0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends[:k]])
    return key, order, offsets


def _places(s):
    """Each slot's place in a (groups, most) table of rows; unassigned slots in a spare last row."""
    k, most = s["groups"], s["most"]
    key, order, offsets = _sorted_rows(s["labels"], k)
    rank = torch.empty_like(order)
    rank[order] = torch.arange(order.numel(), device=order.device)
    place = key * most + (rank - offsets[key])
    return torch.where(key < k, place, torch.full_like(place, k * most)), key


def _spread_rows(rows, place, k, most):
    table = rows.new_zeros(k * most + 1, rows.shape[-1])
    table[place] = rows
    table[-1] = 0
    return table[:-1].view(k, most, -1)


def _take_rows(table, place):
    flat = table.reshape(-1, table.shape[-1])
    return torch.cat([flat, flat.new_zeros(1, flat.shape[-1])])[place]


def _plain_products(s):
    x, w = s["x"].float(), s["weight"].float()
    k, top, most = s["groups"], s["top"], s["most"]
    place, _ = _places(s)
    xt = _spread_rows(x.repeat_interleave(top, 0) if top > 1 else x, place, k, most)
    yt = torch.matmul(xt, w)
    if s["bias"] is not None:
        yt = yt + s["bias"].float()[:, None, :]
    y = _take_rows(yt, place).to(s["x"].dtype).view(*s["labels"].shape, -1)
    if s["op"] == "forward":
        return {"y": y}
    gt = _spread_rows(s["grad"].float().reshape(-1, s["n_out"]), place, k, most)
    gx = _take_rows(torch.matmul(gt, w.transpose(1, 2)), place)
    gx = gx.view(s["rows"], top, -1).sum(1)
    out = {"y": y, "grad_x": gx.to(s["x"].dtype), "grad_weight": torch.matmul(xt.transpose(1, 2), gt).to(s["x"].dtype)}
    if s["bias"] is not None:
        out["grad_bias"] = gt.sum(1).to(s["x"].dtype)
    return out


def _plain_orthogonal(s):
    g = s["update"]
    a, b, c = COEFFICIENTS
    x = g.float()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1) if tall else x
    for _ in range(s["steps"]):
        p = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * p + c * torch.matmul(p, p), x)
    return {"q": (x.transpose(-2, -1) if tall else x).contiguous().to(g.dtype)}


def _plain(s):
    if s["op"] == "route":
        _, order, offsets = _sorted_rows(s["labels"], s["groups"])
        return {"order": order.int(), "offsets": offsets.int()}
    return _plain_orthogonal(s) if s["op"] == "orthogonal" else _plain_products(s)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


def _own(s):
    import gmmxx_b200 as gm

    if s["op"] == "orthogonal":
        return {"q": gm.orthogonalize(s["update"], steps=s["steps"], coefficients=COEFFICIENTS, eps=EPS)}
    groups = gm.group_rows(s["labels"], s["groups"])
    if s["op"] == "route":
        return {"order": groups.order, "offsets": groups.offsets}
    y = gm.grouped_matmul(s["x"], s["weight"], groups, bias=s["bias"])
    if s["op"] == "forward":
        return {"y": y}
    gx, gw, gb = gm.grouped_matmul_backward(s["grad"], s["x"], s["weight"], groups, bias=s["bias"] is not None)
    out = {"y": y, "grad_x": gx, "grad_weight": gw}
    if s["bias"] is not None:
        out["grad_bias"] = gb
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    if case["op"] == "route":
        slots = case["rows"] * case["top"]
        size = 8 if case["index"] == "int64" else 4
        return {"bytes": slots * (size + 4) + 4 * (case["groups"] + 1), "flops": slots}
    size = BYTES[case["dtype"]]
    if case["op"] == "orthogonal":
        lo, hi, b = min(case["m"], case["n"]), max(case["m"], case["n"]), case["batch"]
        # p and p^2 are symmetric: one half of each is enough
        return {"bytes": 2 * size * b * lo * hi, "flops": case["steps"] * b * (3 * lo * lo * hi + lo**3)}
    slots, rows, k = case["rows"] * case["top"], case["rows"], case["groups"]
    n_in, n_out = case["n_in"], case["n_out"]
    used = min(k, slots)  # matrices that some row asks for
    bias = used * n_out if case["bias"] else 0
    moved = size * (rows * n_in + used * n_in * n_out + bias + slots * n_out) + 8 * slots
    flops = 2 * slots * n_in * n_out
    if case["op"] == "step":
        moved += size * (slots * n_out + rows * n_in + k * n_in * n_out + (k * n_out if case["bias"] else 0))
        flops *= 3
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return None  # whole numbers: the plain form's have to be met exactly
    if case["op"] == "orthogonal":
        # p(sigma) of every singular value: U p(S) V^T by the iteration on the Gram matrix of the short side
        g = s["update"].double()
        wide = g if g.shape[-2] <= g.shape[-1] else g.mT
        y = wide / (torch.linalg.matrix_norm(wide)[:, None, None] + EPS)
        total = torch.eye(y.shape[-2], dtype=torch.float64, device=y.device).expand(y.shape[0], -1, -1)
        gram = y @ y.mT
        a, b, c = COEFFICIENTS
        one = total
        for _ in range(case["steps"]):
            # x <- P x with P = a + b G + c G^2, so that G <- P G P, and the steps' P multiply up
            p = a * one + b * gram + c * (gram @ gram)
            total = p @ total
            gram = p @ gram @ p
        q = total @ y
        return {"q": q if g.shape[-2] <= g.shape[-1] else q.mT}
    x, w = s["x"].double(), s["weight"].double()
    flat = s["labels"].reshape(-1)
    top, n_in, n_out = case["top"], case["n_in"], case["n_out"]
    y = x.new_zeros(flat.numel(), n_out)
    gx = x.new_zeros(flat.numel(), n_in)
    gw, gb = torch.zeros_like(w), x.new_zeros(case["groups"], n_out)
    grad = s["grad"].double().reshape(-1, n_out) if case["op"] == "step" else None
    for k in range(case["groups"]):
        slots = torch.nonzero(flat == k).squeeze(1)
        rows = x[slots // top]
        y[slots] = rows @ w[k] + (s["bias"][k].double() if case["bias"] else 0.0)
        if grad is not None:
            gx[slots] = grad[slots] @ w[k].T
            gw[k] = rows.T @ grad[slots]
            gb[k] = grad[slots].sum(0)
    out = {"y": y.view(*s["labels"].shape, n_out)}
    if grad is not None:
        out |= {"grad_x": gx.view(-1, top, n_in).sum(1), "grad_weight": gw}
        if case["bias"]:
            out["grad_bias"] = gb
    return out
