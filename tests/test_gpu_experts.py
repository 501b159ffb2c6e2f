"""The routed products (gmmxx_b200.experts) on the GPU against float64.

Tolerances, derived per element.  A sum of n products held in fp32 is off by
at most n steps of 2^-23 of the sum of the products' magnitudes (one whole
step per addition, which covers an adder that truncates), and splitting fp32
factors into 16-bit planes drops at most 2^-22 of each product; the result is
rounded once to the output's type (half a step, eps / 2 of the value; fp16
below its normal range: half of 2^-24).  Newton-Schulz: see _ns_tolerance."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _close(got, want, mag, n, dtype):
    """|got - want| <= half a step of the type + n steps of the products' magnitude (all float64, CPU)."""
    got = got.double().cpu()
    assert got.shape == want.shape
    tol = (n + 4) * 2.0**-23 * mag
    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)
    if dtype == torch.float16:
        tol = tol + 2.0**-25
    off = (got - want).abs() - tol
    assert not torch.isnan(got).any()
    assert float(off.max()) <= 0 if off.numel() else True, f"off by {float(off.max())} over the tolerance"


def _labels(g, n, top, k, kind):
    shape = (n,) if top == 1 else (n, top)
    if kind == "even":
        return torch.randint(0, k, shape, generator=g)
    if kind == "dropped":  # a third unassigned, by labels on either side
        l = torch.randint(0, k, shape, generator=g)
        u = torch.rand(shape, generator=g)
        return torch.where(u < 0.2, torch.full_like(l, -1), torch.where(u < 0.33, torch.full_like(l, k), l))
    if kind == "one":  # every row to the last component
        return torch.full(shape, k - 1)
    if kind == "none":
        return torch.full(shape, -1)
    assert kind == "skewed"  # one component takes most, many none
    l = torch.randint(0, k, shape, generator=g)
    return torch.where(torch.rand(shape, generator=g) < 0.8, torch.zeros_like(l), l // 2 * 2)


def _reference(x, w, b, labels, gy=None):
    """float64 results and the sums of the products' magnitudes."""
    x, w = x.double().cpu(), w.double().cpu()
    k, n_in, n_out = w.shape
    n = x.shape[0]
    flat = labels.reshape(n, -1)
    top = flat.shape[1]
    out = {"y": torch.zeros(n, top, n_out, dtype=torch.float64)}
    mag = {"y": out["y"].clone()}
    if gy is not None:
        gy = gy.double().cpu().reshape(n, top, n_out)
        for name, shape in (("gx", (n, n_in)), ("gw", (k, n_in, n_out)), ("gb", (k, n_out))):
            out[name], mag[name] = torch.zeros(shape, dtype=torch.float64), torch.zeros(shape, dtype=torch.float64)
    for c in range(k):
        for t in range(top):
            r = torch.nonzero(flat[:, t] == c).squeeze(1)
            if not r.numel():
                continue
            out["y"][r, t] = x[r] @ w[c]
            mag["y"][r, t] = x[r].abs() @ w[c].abs()
            if b is not None:
                out["y"][r, t] += b[c].double().cpu()
                mag["y"][r, t] += b[c].double().cpu().abs()
            if gy is not None:
                out["gx"][r] += gy[r, t] @ w[c].T
                mag["gx"][r] += gy[r, t].abs() @ w[c].abs().T
                out["gw"][c] += x[r].T @ gy[r, t]
                mag["gw"][c] += x[r].abs().T @ gy[r, t].abs()
                out["gb"][c] += gy[r, t].sum(0)
                mag["gb"][c] += gy[r, t].abs().sum(0)
    return out, mag


def _case(dev, n, top, k, n_in, n_out, dtype, kind="even", seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    labels = _labels(g, n, top, k, kind)
    x = torch.randn(n, n_in, generator=g).to(dtype)
    w = (torch.randn(k, n_in, n_out, generator=g) / n_in**0.5).to(dtype)
    b = torch.randn(k, n_out, generator=g).to(dtype) if bias else None
    gy = torch.randn(*labels.shape, n_out, generator=g).to(dtype)
    return [t if t is None else t.to(dev) for t in (labels, x, w, b, gy)]


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------


def _check_groups(labels, k, groups):
    flat = labels.reshape(-1).cpu().long()
    key = torch.where((flat >= 0) & (flat < k), flat, torch.full_like(flat, k))
    want = torch.argsort(key, stable=True)
    assert torch.equal(groups.order.cpu().long(), want)
    counts = torch.bincount(key, minlength=k + 1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)[:k]])
    assert torch.equal(groups.offsets.cpu().long(), offsets)
    # the tile tables cover every position once, in order, within the groups
    t = groups.tiles.cpu().long()
    at = 4
    for i, per in enumerate((128, 256)):
        rows = t[at:at + 3 * int(t[i])].reshape(-1, 3)
        assert torch.equal(rows[:, 1], torch.cat([torch.zeros(1, dtype=torch.int64), rows[:, 2].cumsum(0)])[:-1])
        assert int(rows[:, 2].sum()) == flat.numel()
        if flat.numel():
            assert torch.equal(key[want][rows[:, 1]], rows[:, 0])
            assert torch.equal(key[want][rows[:, 1] + rows[:, 2] - 1], rows[:, 0])
            assert int(rows[:, 2].min()) >= 1 and int(rows[:, 2].max()) <= per
        at += 3 * (flat.numel() // per + min(k + 1, flat.numel()))


@pytest.mark.parametrize("n,top,k", [(1, 1, 1), (31, 1, 3), (129, 2, 16), (4097, 8, 64), (32768, 1, 1500),
                                     (32769, 1, 7), (100003, 1, 8192), (70001, 2, 16384), (300000, 1, 1),
                                     (1000, 1, 16384), (900001, 1, 300), (1500007, 1, 3000), (2, 1, 9000)])
@pytest.mark.parametrize("kind", ["even", "dropped", "skewed"])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_group_rows(cuda_device, n, top, k, kind, dtype):
    import gmmxx_b200 as gm

    labels = _labels(torch.Generator().manual_seed(n), n, top, k, kind).to(dtype).to(cuda_device)
    groups = gm.group_rows(labels, k)
    assert groups.shape == tuple(labels.shape) and groups.n_rows == n and groups.top_k == top
    _check_groups(labels, k, groups)


@pytest.mark.parametrize("kind", ["one", "none"])
@pytest.mark.parametrize("n", [0, 1, 500, 40000])
def test_group_rows_of_one_component_or_none(cuda_device, kind, n):
    import gmmxx_b200 as gm

    labels = _labels(torch.Generator(), n, 1, 5, kind).to(cuda_device)
    _check_groups(labels, 5, gm.group_rows(labels, 5))


def test_group_rows_far_labels(cuda_device):
    """64-bit labels whose low 32 bits are a valid component are unassigned."""
    import gmmxx_b200 as gm

    labels = torch.tensor([1, (1 << 32) + 1, -(1 << 32), -(1 << 63), (1 << 63) - 1, 0], device=cuda_device)
    groups = gm.group_rows(labels, 3)
    assert groups.order.tolist() == [5, 0, 1, 2, 3, 4] and groups.offsets.tolist() == [0, 1, 2, 2]


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------

SHAPES = [
    # n, top, k, n_in, n_out, kind
    (1, 1, 1, 1, 1, "even"),
    (7, 1, 3, 5, 9, "even"),
    (33, 2, 4, 64, 64, "even"),
    (130, 1, 2, 32, 48, "one"),
    (300, 1, 5, 100, 77, "dropped"),
    (257, 3, 7, 65, 130, "skewed"),
    (1000, 1, 9, 128, 256, "dropped"),
    (513, 2, 6, 200, 264, "skewed"),
    (2000, 1, 300, 24, 40, "even"),
    (128, 1, 2, 520, 8, "even"),
    (64, 1, 4, 8, 520, "none"),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,top,k,n_in,n_out,kind", SHAPES)
def test_products_and_gradients(cuda_device, n, top, k, n_in, n_out, kind, dtype):
    import gmmxx_b200 as gm

    labels, x, w, b, gy = _case(cuda_device, n, top, k, n_in, n_out, dtype, kind)
    groups = gm.group_rows(labels, k)
    y = gm.grouped_matmul(x, w, groups, bias=b)
    gx, gw, gb = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)
    ref, mag = _reference(x, w, b, labels.cpu(), gy)
    assert y.dtype == gx.dtype == gw.dtype == gb.dtype == dtype and y.shape == (*labels.shape, n_out)
    most = max(1, int((groups.offsets[1:] - groups.offsets[:-1]).max()))
    _close(y.reshape(n, top, n_out), ref["y"], mag["y"], n_in + 1, dtype)
    _close(gx, ref["gx"], mag["gx"], n_out + top, dtype)
    _close(gw, ref["gw"], mag["gw"], most, dtype)
    _close(gb, ref["gb"], mag["gb"], most, dtype)
    if kind in ("dropped", "none"):
        lost = ((labels < 0) | (labels >= k)).cpu()
        assert not y.cpu()[lost].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,top,k,n_in,n_out,kind", [(6000, 1, 5, 136, 1000, "skewed"), (5000, 2, 3, 264, 776, "dropped"),
                                                     (20000, 1, 4, 520, 300, "even")])
def test_pairs_of_blocks(cuda_device, n, top, k, n_in, n_out, kind, dtype):
    """Sizes whose products run on pairs of blocks: ragged last tiles, columns
    and contractions that are no multiple of anything."""
    import gmmxx_b200 as gm

    labels, x, w, b, gy = _case(cuda_device, n, top, k, n_in, n_out, dtype, kind)
    groups = gm.group_rows(labels, k)
    y = gm.grouped_matmul(x, w, groups, bias=b)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    gx, gw, gb = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)
    hx, hw, _ = gm.grouped_matmul_backward(gy, x, wt, groups)
    ref, mag = _reference(x, w, b, labels.cpu(), gy)
    most = int((groups.offsets[1:] - groups.offsets[:-1]).max())
    _close(y.reshape(n, top, n_out), ref["y"], mag["y"], n_in + 1, dtype)
    _close(gm.grouped_matmul(x, wt, groups, bias=b).reshape(n, top, n_out), ref["y"], mag["y"], n_in + 1, dtype)
    for got in ((gx, gw), (hx, hw)):
        _close(got[0], ref["gx"], mag["gx"], n_out + top, dtype)
        _close(got[1], ref["gw"], mag["gw"], most, dtype)
    _close(gb, ref["gb"], mag["gb"], most, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,top,k,n_in,n_out,kind", [(30, 1, 9, 1100, 132, "even"), (37, 2, 20, 2051, 36, "dropped"),
                                                     (20, 2, 11, 2052, 37, "dropped"),
                                                     (140, 1, 36, 70, 1028, "skewed"), (50, 1, 16, 4, 300, "one")])
def test_few_rows_per_group(cuda_device, n, top, k, n_in, n_out, kind, dtype):
    """Groups of a few rows (and one of many), contractions longer than what is
    staged at a time, both orders of the weights."""
    import gmmxx_b200 as gm

    labels, x, w, b, gy = _case(cuda_device, n, top, k, n_in, n_out, dtype, kind)
    groups = gm.group_rows(labels, k)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    ref, mag = _reference(x, w, b, labels.cpu(), gy)
    most = max(1, int((groups.offsets[1:] - groups.offsets[:-1]).max()))
    for weight in (w, wt):
        y = gm.grouped_matmul(x, weight, groups, bias=b)
        gx, gw, gb = gm.grouped_matmul_backward(gy, x, weight, groups, bias=True)
        _close(y.reshape(n, top, n_out), ref["y"], mag["y"], n_in + 1, dtype)
        _close(gx, ref["gx"], mag["gx"], n_out + top, dtype)
        _close(gw, ref["gw"], mag["gw"], most, dtype)
        _close(gb, ref["gb"], mag["gb"], most, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_groups(cuda_device, dtype):
    """Groups of tens of thousands of rows: the weight gradient's sum is split and joined."""
    import gmmxx_b200 as gm

    labels, x, w, b, gy = _case(cuda_device, 90001, 1, 3, 40, 56, dtype, "skewed")
    groups = gm.group_rows(labels, 3)
    y = gm.grouped_matmul(x, w, groups, bias=b)
    gx, gw, gb = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)
    ref, mag = _reference(x, w, b, labels.cpu(), gy)
    most = int((groups.offsets[1:] - groups.offsets[:-1]).max())
    _close(y[:, None], ref["y"], mag["y"], 41, dtype)
    _close(gx, ref["gx"], mag["gx"], 56, dtype)
    _close(gw, ref["gw"], mag["gw"], most, dtype)
    _close(gb, ref["gb"], mag["gb"], most, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_in,n_out", [(64, 96), (37, 50)])
def test_transposed_and_strided_inputs(cuda_device, dtype, n_in, n_out):
    """A transposed weight is read in place and its gradient comes in its
    order; rows cut out of wider ones give the same bits as their copies."""
    import gmmxx_b200 as gm

    labels, x, w, b, gy = _case(cuda_device, 200, 1, 5, n_in, n_out, dtype)
    groups = gm.group_rows(labels, 5)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    y, yt = gm.grouped_matmul(x, w, groups, b), gm.grouped_matmul(x, wt, groups, b)
    assert torch.equal(y, yt)
    g, gt = gm.grouped_matmul_backward(gy, x, w, groups), gm.grouped_matmul_backward(gy, x, wt, groups)
    assert gt[1].stride() == wt.stride() and g[2] is None
    ref, mag = _reference(x, w, b, labels.cpu(), gy)
    for got in (g, gt):
        _close(got[0], ref["gx"], mag["gx"], n_out, dtype)
        _close(got[1], ref["gw"], mag["gw"], 200, dtype)
    wide = torch.zeros(200, n_in + 3, dtype=dtype, device=cuda_device)
    wide[:, 2:2 + n_in] = x
    assert torch.equal(gm.grouped_matmul(wide[:, 2:2 + n_in], w, groups, b), y)
    shifted = torch.empty(w.numel() + 1, dtype=dtype, device=cuda_device)[1:].view_as(w)  # off any 16-byte boundary
    shifted.copy_(w)
    xs = torch.empty(x.numel() + 1, dtype=dtype, device=cuda_device)[1:].view_as(x)
    xs.copy_(x)
    assert torch.equal(gm.grouped_matmul(xs, shifted, groups, b), y)


def test_parts_of_the_backward(cuda_device):
    import gmmxx_b200 as gm

    labels, x, w, b, gy = _case(cuda_device, 100, 2, 4, 40, 24, torch.float32)
    groups = gm.group_rows(labels, 4)
    whole = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)
    for i, kw in enumerate((dict(need_weight=False), dict(need_x=False), dict(need_x=False, need_weight=False, bias=True))):
        part = gm.grouped_matmul_backward(gy, x, w, groups, **kw)
        for j in range(3):
            assert part[j] is None if j != i else torch.equal(part[j], whole[j])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_of_one_component_stay_there(cuda_device, dtype):
    """Infinities and NaN in one component's rows, weights and gradients (and
    in unassigned rows) reach no other component."""
    import gmmxx_b200 as gm

    n, k, n_in, n_out = 700, 6, 72, 80
    labels, x, w, b, gy = _case(cuda_device, n, 1, k, n_in, n_out, dtype, "dropped")
    groups = gm.group_rows(labels, k)
    y0 = gm.grouped_matmul(x, w, groups, b)
    g0 = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)
    bad = (labels == 2) | (labels < 0) | (labels >= k)
    x[bad], gy[bad], w[2] = float("nan"), float("inf"), float("nan")
    y1 = gm.grouped_matmul(x, w, groups, b)
    g1 = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)
    keep = torch.tensor([c for c in range(k) if c != 2], device=cuda_device)
    assert torch.equal(y0[~bad], y1[~bad])
    lost = (labels < 0) | (labels >= k)
    assert not y1[lost].any() and not g1[0][lost].any()
    assert torch.equal(g0[0][~bad], g1[0][~bad])
    assert torch.equal(g0[1][keep], g1[1][keep]) and torch.equal(g0[2][keep], g1[2][keep])
    assert torch.isnan(y1[labels == 2]).all() and torch.isnan(g1[1][2]).all() and torch.isinf(g1[2][2]).all()


def test_gradients_against_differences(cuda_device):
    """The products are linear in x, w and b: a step of any size gives the
    derivative up to rounding.  fp32, sum over outputs weighted by gy."""
    import gmmxx_b200 as gm

    labels, x, w, b, gy = _case(cuda_device, 90, 2, 4, 33, 21, torch.float32, "dropped")
    groups = gm.group_rows(labels, 4)
    gx, gw, gb = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)

    def loss(x, w, b):
        return (gm.grouped_matmul(x, w, groups, b).double() * gy.double()).sum()

    gen = torch.Generator(device=cuda_device).manual_seed(5)
    dx, dw, db = (torch.randn(t.shape, generator=gen, device=cuda_device) for t in (x, w, b))
    for moved, grad, step in (((x + dx, w, b), gx, dx), ((x, w + dw, b), gw, dw), ((x, w, b + db), gb, db)):
        got = loss(*moved) - loss(x, w, b)
        want = (grad.double() * step.double()).sum()
        # 33-term sums of magnitude ~10 (w + dw is O(1) per term) in fp32, 180 x 21 outputs: 1e-5 of each at most
        scale = (gm.grouped_matmul(moved[0].abs(), moved[1].abs(), groups, moved[2].abs()).double() * gy.abs().double()).sum()
        assert abs(float(got - want)) <= 37 * 2.0**-22 * float(scale)


def test_empty_calls(cuda_device):
    import gmmxx_b200 as gm

    labels = torch.empty(0, dtype=torch.int64, device=cuda_device)
    groups = gm.group_rows(labels, 3)
    x, w = torch.empty(0, 8, device=cuda_device), torch.randn(3, 8, 4, device=cuda_device)
    assert gm.grouped_matmul(x, w, groups).shape == (0, 4)
    gx, gw, gb = gm.grouped_matmul_backward(torch.empty(0, 4, device=cuda_device), x, w, groups, bias=True)
    assert gx.shape == (0, 8) and not gw.any() and not gb.any() and gw.shape == w.shape
    assert gm.orthogonalize(torch.empty(0, 3, 4, device=cuda_device)).shape == (0, 3, 4)


# ---------------------------------------------------------------------------
# Newton-Schulz
# ---------------------------------------------------------------------------


def _ns(g, steps, coef, eps, dtype):
    a, b, c = coef
    x = g.to(dtype)
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt().to(dtype) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        p = x @ x.mT
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.mT if tall else x


def _ns_check(q, g, steps=5, coef=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """In norm, per matrix: the kernel rounds the iterates where a float32
    iteration rounds them.  Two fp16 planes (fp32 and fp16 results, and bf16
    ones of short sides below 256 or more than 6 steps) keep 2^-23 where float32 keeps 2^-24, drop
    products of 2^-22 and add with truncation: 8 times a float32 iteration's
    own distance from float64 (with a floor of 4 steps of 2^-24, where the float32
    iteration happens to be exact).  One fp16 plane (bf16 results, larger)
    keeps 2^-12: 2^12 times that, times 2.  Then the result's own rounding."""
    ref = _ns(g.cpu(), steps, coef, eps, torch.float64)
    own = _ns(g.float().cpu(), steps, coef, eps, torch.float32).double()
    norm = ref.flatten(-2).norm(dim=-1)
    off32 = (own - ref).flatten(-2).norm(dim=-1).clamp_min(1e-300) + 4 * 2.0**-24 * norm
    one_plane = g.dtype == torch.bfloat16 and min(g.shape[-2:]) >= 256 and steps <= 6
    tol = (8192 if one_plane else 8) * off32 + torch.finfo(g.dtype).eps / 2 * norm
    if g.dtype == torch.float16:
        tol = tol + 2.0**-25 * (g.shape[-1] * g.shape[-2]) ** 0.5
    off = (q.double().cpu() - ref).flatten(-2).norm(dim=-1)
    assert q.dtype == g.dtype and q.shape == g.shape
    assert bool((off <= tol).all()), (off / norm, tol / norm)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 1, 9), (2, 5, 3), (4, 64, 64), (3, 33, 100), (2, 130, 64),
                                   (1, 128, 128), (2, 129, 200), (1, 300, 257), (2, 256, 520), (1, 520, 256),
                                   (24, 520, 776), (20, 1000, 536), (1, 135, 1500), (2, 2000, 140), (1, 259, 900), (3, 60, 500), (2, 90, 250), (2, 250, 100),
                                   (260, 16, 16), (2, 3, 24, 40)])
def test_orthogonalize(cuda_device, shape, dtype):
    import gmmxx_b200 as gm

    g = torch.Generator().manual_seed(sum(shape))
    m = (torch.randn(*shape, generator=g) * torch.exp(torch.randn(*shape[:-1], 1, generator=g)) * 0.01).to(dtype)
    _ns_check(gm.orthogonalize(m.to(cuda_device)).cpu(), m)


@pytest.mark.parametrize("steps", [0, 1, 2, 8])
@pytest.mark.parametrize("shape", [(2, 40, 56), (1, 200, 140)])
def test_orthogonalize_steps_and_coefficients(cuda_device, steps, shape):
    import gmmxx_b200 as gm

    m = torch.randn(*shape, generator=torch.Generator().manual_seed(steps))
    _ns_check(gm.orthogonalize(m.to(cuda_device), steps=steps).cpu(), m, steps)
    cubic = (1.5, -0.5, 0.0)
    _ns_check(gm.orthogonalize(m.to(cuda_device), steps=steps, coefficients=cubic, eps=1e-3).cpu(), m, steps, cubic, 1e-3)


@pytest.mark.parametrize("steps", [6, 7, 12])
def test_orthogonalize_many_steps_in_bf16(cuda_device, steps):
    import gmmxx_b200 as gm

    m = torch.randn(1, 270, 400, generator=torch.Generator().manual_seed(steps)).to(torch.bfloat16)
    _ns_check(gm.orthogonalize(m.to(cuda_device), steps=steps).cpu(), m, steps)


def test_orthogonalize_extremes(cuda_device):
    """Zero, tiny and huge matrices, a rank-one one, a transposed view."""
    import gmmxx_b200 as gm

    g = torch.Generator().manual_seed(3)
    base = torch.randn(6, 48, 80, generator=g)
    base[1] = 0
    base[2] *= 1e-30
    base[3] *= 1e30  # the sum of squares is beyond float32
    base[4] = base[4, :, :1] * base[4, :1, :]
    q = gm.orthogonalize(base.to(cuda_device)).cpu()
    assert not q[1].any()
    keep = [0, 3, 4, 5]
    _ns_check(q[keep], base[keep])
    assert float(q[2].abs().max()) < 1e-18  # |g| far below eps stays small: 484 * 6e-29 / 1e-7
    v = base[0].mT.to(cuda_device)
    assert torch.equal(gm.orthogonalize(v), gm.orthogonalize(v.contiguous()))
    bad = base[:3].clone()
    bad[0, 3, 5] = float("nan")
    q2 = gm.orthogonalize(bad.to(cuda_device)).cpu()
    assert torch.isnan(q2[0]).all() and not torch.isnan(q2[1:]).any()


# ---------------------------------------------------------------------------
# together, and how calls share the device
# ---------------------------------------------------------------------------


def _step(gm, labels, x, w, b, gy, k):
    groups = gm.group_rows(labels, k)
    y = gm.grouped_matmul(x, w, groups, b)
    gx, gw, gb = gm.grouped_matmul_backward(gy, x, w, groups, bias=True)
    return (groups.order, y, gx, gw, gb, gm.orthogonalize(gw))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_repeated_streamed_and_captured_calls_give_the_same_bits(cuda_device, dtype):
    import gmmxx_b200 as gm

    args = _case(cuda_device, 3000, 2, 8, 96, 160, dtype, "dropped")
    want = _step(gm, *args, 8)
    for a, b in zip(want, _step(gm, *args, 8)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(gm, *args, 8)
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    # two captured graphs, replayed at the same time on two streams with new inputs in place
    other = _case(cuda_device, 3000, 2, 8, 96, 160, dtype, "skewed", seed=9)
    want_other = _step(gm, *other, 8)
    bufs = [[t.clone() for t in args], [t.clone() for t in args]]
    graphs, outs = [], []
    for buf in bufs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(gm, *buf, 8))
        graphs.append(graph)
    for buf, src in zip(bufs, (other, args)):
        for d, s in zip(buf, src):
            d.copy_(s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for want_i, out in zip((want_other, want), outs):
        for a, b in zip(want_i, out):
            assert torch.equal(a, b)


def test_a_mixture_routes_its_rows_to_learned_maps(cuda_device):
    """Fit, predict, and learn each component's rotation from its rows: the
    labels of a fitted mixture route the rows; the orthogonalised correlation
    of a component's rows with their rotated images gives its rotation back."""
    import gmmxx_b200 as gm

    k, d, n = 4, 16, 20000
    g = torch.Generator().manual_seed(11)
    centers = torch.randn(k, d, generator=g) * 8
    comp = torch.randint(0, k, (n,), generator=g)
    x = (centers[comp] + torch.randn(n, d, generator=g)).to(cuda_device)
    model = gm.GMMXX(n_components=k, covariance_type="diag", max_iter=20).fit(x)
    labels = model.predict(x)
    groups = gm.group_rows(labels, k)
    counts = groups.offsets[1:] - groups.offsets[:-1]
    assert int(counts.sum()) == n and torch.equal(counts.long(), torch.bincount(labels, minlength=k))
    rot = torch.linalg.qr(torch.randn(k, d, d, generator=g))[0].to(cuda_device)
    # sums per component: the weight gradient of all-ones rows
    ones = torch.ones(n, 1, device=cuda_device)
    mean = gm.grouped_matmul_backward(x, ones, torch.zeros(k, 1, d, device=cuda_device), groups, need_x=False)[1]
    mean = mean[:, 0] / counts[:, None]
    white = gm.grouped_matmul(ones, -mean[:, None, :].contiguous(), groups) + x
    image = gm.grouped_matmul(white, rot, groups)
    corr = gm.grouped_matmul_backward(image, white, rot, groups, need_x=False)[1]
    # corr = S rot with S close to n_k I: its polar factor is close to rot; the cubic converges to it
    q = gm.orthogonalize(corr, steps=30, coefficients=(1.5, -0.5, 0.0))
    eye = torch.eye(d, device=cuda_device)
    # converged: q q^T = 1 up to the iterates' rounding (2^-23 each of d terms and 30 steps, not adding up
    # because every step corrects: 64 steps of 2^-23)
    assert float((q @ q.mT - eye).abs().max()) < 64 * 2.0**-23
    s = image.double()
    u, _, vh = torch.linalg.svd(corr.double())
    assert float((q.double() - u @ vh).norm(dim=(1, 2)).max()) < 1e-3  # sigma spread below 2: conditioning ~1
    assert s.isfinite().all()
