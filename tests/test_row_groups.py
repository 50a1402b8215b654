"""Rows in groups (tfh_group_rows, tfh_ragged_gemm*, tfh_combine_rows*, tfh_adapter_gemm*): against plain loops in 64 bits
on the CPU, at the sizes, layouts and groups where such kernels go wrong, and what the entry points refuse.

Tolerances, element by element, from arithmetic alone: a result is rounded once (half a step of its type relative to it, or
half the smallest step of f16 where that is larger), and a sum of k products held in f32 (f64) is off by at most
2 (k + 4) u times the sum of the products' absolute values, u = 2^-24 (2^-53).  The adapters' middle X A is kept to at
least 16 bits (half a step 2^-17) beside 16-bit operands."""
import ctypes as C
import itertools
import os

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def tf():
    import tenferro_rs_amd as tf
    tf.lib()
    return tf


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch


TYPES = ["bfloat16", "float16", "float32", "float64"]
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24, "float64": 2.0 ** -53}
U = {"bfloat16": 2.0 ** -24, "float16": 2.0 ** -24, "float32": 2.0 ** -24, "float64": 2.0 ** -53}
SMALLEST = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -150, "float64": 0.0}
MIDDLE = {"bfloat16": 2.0 ** -17, "float16": 2.0 ** -17, "float32": 0.0, "float64": 0.0}


def close(got, want, size, k, name, extra=0.0):
    """`size`: the sum of the products' absolute values; `extra`: further absolute slack, derived by the caller."""
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    bound = HALF_STEP[name] * (1 + 2 ** -6) * want.abs() + SMALLEST[name] + 2 * (k + 4) * U[name] * size.double().cpu() + extra
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (name, int(bad.sum()), off[bad][:4].tolist(), bound[bad][:4].tolist(), bad.nonzero()[:4].tolist())


def grouping(ids, n):
    """offsets, order, positions of a flat list of indices, in plain Python."""
    ids = [int(i) for i in ids]
    order = [i for g in range(n) for i, x in enumerate(ids) if x == g]
    grouped = len(order)
    order += [i for i, x in enumerate(ids) if not 0 <= x < n]
    offsets = [0]
    for g in range(n):
        offsets.append(offsets[-1] + sum(1 for x in ids if x == g))
    positions = [-1] * len(ids)
    for p in range(grouped):
        positions[order[p]] = p
    return offsets, order, positions


def choices(rng, tokens, fan, groups, none=0.15, only=None):
    """Distinct choices for each token; `only`: groups that are chosen at all (the others stay empty)."""
    pool = np.arange(groups) if only is None else np.asarray(only)
    ids = np.stack([rng.permutation(pool)[:fan] if len(pool) >= fan else rng.choice(pool, fan) for _ in range(tokens)]) if tokens else np.zeros((0, fan), int)
    ids = np.where(rng.random(ids.shape) < none, rng.choice([-1, groups, groups + 7, -5], ids.shape), ids)
    return ids


def made(tf, torch, ids, groups):
    return tf.RowGroups.from_ids(torch.from_numpy(np.ascontiguousarray(ids)).cuda(), groups)


def tensor(torch, rng, shape, name, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(getattr(torch, name))


def layout(torch, t, how):
    """The same values on the GPU with other strides."""
    t = t.cuda()
    if how == "columns":        # the last axis contiguous
        return t.contiguous()
    if how == "rows":           # the last but one contiguous
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)
    if how == "pitch":          # rows further apart than they are long, and an odd start
        big = torch.zeros(*t.shape[:-2], t.shape[-2] + 1, t.shape[-1] + 3, dtype=t.dtype, device="cuda")
        view = big[..., 1:, 1:t.shape[-1] + 1]
        view.copy_(t)
        return view
    if how == "steps":          # every second element of both axes
        big = torch.zeros(*t.shape[:-2], 2 * t.shape[-2], 2 * t.shape[-1], dtype=t.dtype, device="cuda")
        view = big[..., ::2, ::2]
        view.copy_(t)
        return view
    raise ValueError(how)


# ------------------------------------------------------------------------------------------------------ grouping
GROUPINGS = [(0, 1, 3), (1, 1, 1), (1, 8, 9), (5, 1, 2048), (63, 1, 2), (64, 3, 3), (257, 4, 65), (1000, 2, 7), (1024, 8, 128),
             (2731, 3, 512), (8192, 1, 2), (8193, 1, 2), (5000, 8, 64), (70001, 2, 2047)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,fan,groups", GROUPINGS)
@pytest.mark.parametrize("bits", [32, 64])
def test_grouping_is_the_stable_one(tf, torch, tokens, fan, groups, bits):
    rng = np.random.default_rng(tokens + groups)
    ids = rng.integers(-1, groups + 1, (tokens, fan)).astype(np.int32 if bits == 32 else np.int64)
    g = made(tf, torch, ids, groups)
    key = np.where((ids >= 0) & (ids < groups), ids, groups).reshape(-1)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(groups + 1))
    positions = np.empty(len(key), int)
    positions[order] = np.arange(len(key))
    positions[key == groups] = -1
    assert g.n_rows == tokens * fan and g.n_groups == groups and (g.fan == fan)
    assert g.offsets.cpu().numpy().tolist() == offsets.tolist()
    assert np.array_equal(g.order.cpu().numpy(), order)
    assert np.array_equal(g.positions.cpu().numpy(), positions)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["all one", "all none", "last only", "huge 64-bit"])
def test_grouping_of_extreme_indices(tf, torch, how):
    n, groups = 9000, 33
    ids = np.zeros(n, np.int64)
    if how == "all none":
        ids[:] = -1
    elif how == "last only":
        ids[:] = groups - 1
    elif how == "huge 64-bit":       # their low halves are valid indices
        ids[:] = np.where(np.arange(n) % 2 == 0, (1 << 32) + 5, -(1 << 40) + 3)
    g = made(tf, torch, ids, groups)
    offsets, order, positions = grouping(ids, groups)
    assert g.offsets.tolist() == offsets and g.order.tolist() == order and g.positions.tolist() == positions


@pytest.mark.gpu
def test_grouping_reads_strided_indices(tf, torch):
    rng = np.random.default_rng(3)
    base = torch.from_numpy(rng.integers(0, 6, (40, 10))).cuda()
    for view in (base[:, 2:5], base.t()[1:4].t(), base[::3, ::4], base[:, 7], base[5], base[3:4, 1:8:2], base[:, 1:2], base[:1, 4:5].expand(9, 3)):
        g = tf.RowGroups.from_ids(view, 6)
        offsets, order, positions = grouping(view.reshape(-1).cpu().numpy(), 6)
        assert g.offsets.tolist() == offsets and g.order.tolist() == order and g.positions.tolist() == positions


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,fan,groups", [(1025, 1, 3), (150000, 2, 256), (16385, 1, 319), (20000, 1, 320), (300000, 1, 2048)])
def test_grouping_of_many_rows(tf, torch, tokens, fan, groups):
    rng = np.random.default_rng(groups)
    ids = torch.from_numpy(rng.integers(-1, groups + 1, (tokens, fan))).cuda()
    g = tf.RowGroups.from_ids(ids, groups)
    flat = torch.where((ids.reshape(-1) < 0) | (ids.reshape(-1) >= groups), groups, ids.reshape(-1))
    key, order = torch.sort(flat, stable=True)
    positions = torch.empty_like(order)
    positions[order] = torch.arange(len(order), device="cuda")
    assert torch.equal(g.order.long(), order)
    assert torch.equal(g.offsets.long(), torch.searchsorted(key, torch.arange(groups + 1, device="cuda")))
    assert torch.equal(g.positions.long(), torch.where(flat < groups, positions, -1))


# ------------------------------------------------------------------------------------------------------ products
def ragged_reference(torch, a, b, offsets, order, fan, gather):
    """c and the sums of absolute values, zeros for rows of no group."""
    n = len(order)
    a, b = a.double(), b.double()
    c, size = torch.zeros(n, b.shape[2], dtype=torch.float64), torch.zeros(n, b.shape[2], dtype=torch.float64)
    for g in range(len(offsets) - 1):
        for p in range(offsets[g], offsets[g + 1]):
            row = a[order[p] // fan if gather else p]
            c[p], size[p] = row @ b[g], row.abs() @ b[g].abs()
    return c, size


SHAPES = [  # tokens, fan, groups, K, N
    (1, 1, 1, 1, 1), (1, 2, 3, 8, 16), (7, 1, 5, 33, 5), (16, 4, 8, 64, 64), (40, 2, 3, 129, 65), (130, 3, 4, 72, 200), (300, 1, 2, 256, 136),
    (65, 2, 70, 40, 24), (3, 2, 2, 520, 264), (200, 2, 3, 1000, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("how", ["columns", "rows"])
@pytest.mark.parametrize("gather", [False, True])
def test_ragged_product(tf, torch, name, shape, how, gather):
    tokens, fan, groups, K, N = shape
    rng = np.random.default_rng(tokens * 7 + K)
    ids = choices(rng, tokens, min(fan, groups), groups)
    fan = ids.shape[1]
    offsets, order, _ = grouping(ids.reshape(-1), groups)
    a = tensor(torch, rng, (tokens if gather else tokens * fan, K), name)
    b = tensor(torch, rng, (groups, K, N), name, K ** -0.5)
    want, size = ragged_reference(torch, a, b, offsets, order, fan, gather)
    got = tf.ragged_gemm(a.cuda(), layout(torch, b, how), made(tf, torch, ids, groups), gather=gather)
    close(got, want, size, K, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16", "float64"])
@pytest.mark.parametrize("how_a,how_b,how_c", [("pitch", "pitch", "pitch"), ("rows", "steps", "columns"), ("steps", "columns", "rows"), ("columns", "rows", "steps")])
def test_ragged_product_into_strided_views(tf, torch, name, how_a, how_b, how_c):
    rng = np.random.default_rng(11)
    tokens, fan, groups, K, N = 90, 2, 5, 88, 72
    ids = choices(rng, tokens, fan, groups, only=[0, 3])           # three groups are empty
    offsets, order, _ = grouping(ids.reshape(-1), groups)
    a, b, c = (tensor(torch, rng, s, name) for s in ((tokens, K), (groups, K, N), (tokens * fan, N)))
    want, size = ragged_reference(torch, a, b, offsets, order, fan, True)
    grouped = offsets[-1]
    want = 0.5 * want - 1.5 * c.double()
    want[grouped:] = c.double()[grouped:]
    size = 0.5 * size + 1.5 * c.double().abs()
    out = layout(torch, c, how_c)
    tf.ragged_gemm_into(layout(torch, a, how_a), layout(torch, b, how_b), made(tf, torch, ids, groups), 0.5, -1.5, out, gather=True)
    close(out, want, size, K, name)
    assert torch.equal(out.cpu()[grouped:], c[grouped:])           # rows of no group stay as they were


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
def test_ragged_product_scatters_and_overwrites_what_is_no_number(tf, torch, name):
    rng = np.random.default_rng(5)
    tokens, fan, groups, K, N = 50, 3, 4, 64, 40
    ids = choices(rng, tokens, fan, groups)
    offsets, order, _ = grouping(ids.reshape(-1), groups)
    a, b = tensor(torch, rng, (tokens * fan, K), name), tensor(torch, rng, (groups, K, N), name)
    want, size = ragged_reference(torch, a, b, offsets, order, fan, False)
    out = torch.full((tokens * fan, N), float("nan"), dtype=a.dtype, device="cuda")
    tf.ragged_gemm_into(a.cuda(), b.cuda(), made(tf, torch, ids, groups), 1.0, 0.0, out, scatter=True)
    kept = torch.tensor(order[:offsets[-1]])
    close(out.cpu()[kept], want[:offsets[-1]], size[:offsets[-1]], K, name)
    assert out.cpu()[torch.tensor(order[offsets[-1]:], dtype=torch.long)].isnan().all()


@pytest.mark.gpu
def test_ragged_product_without_rows_groups_or_k(tf, torch):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    g = tf.RowGroups.from_ids(torch.zeros(0, dtype=torch.int32, device="cuda"), 4)
    assert g.offsets.tolist() == [0] * 5
    assert tf.ragged_gemm(z(0, 8), z(4, 8, 6), g).shape == (0, 6)
    da, db = tf.ragged_gemm_backward(z(0, 8), torch.ones(4, 8, 6, dtype=torch.bfloat16, device="cuda"), z(0, 6), g)
    assert da.shape == (0, 8) and db.shape == (4, 8, 6) and not db.any()
    g = tf.RowGroups.from_ids(torch.tensor([1, -1, 0], device="cuda"), 2)
    out = tf.ragged_gemm(z(3, 0), z(2, 0, 5), g)                    # nothing to sum: zeros
    assert out.shape == (3, 5) and not out.any()
    assert tf.ragged_gemm(z(3, 4), z(2, 4, 0), g).shape == (3, 0)
    none = tf.RowGroups.from_ids(torch.full((3,), -1, device="cuda"), 2)
    out = tf.ragged_gemm(torch.ones(3, 4, dtype=torch.bfloat16, device="cuda"), torch.ones(2, 4, 5, dtype=torch.bfloat16, device="cuda"), none)
    assert not out.any()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float32"])
def test_ragged_product_keeps_infinities_to_their_groups_and_rows(tf, torch, name):
    rng = np.random.default_rng(8)
    ids = np.array([0, 1, 1, 2, 2, 2, -1, 0])
    a, b = tensor(torch, rng, (8, 48), name), tensor(torch, rng, (3, 48, 32), name)
    clean = tf.ragged_gemm(a.cuda(), b.cuda(), made(tf, torch, ids, 3), gather=True).cpu()
    b[1] = float("inf")
    a[6] = float("nan")                                           # the row of no group
    a[0, 3] = float("nan")
    got = tf.ragged_gemm(a.cuda(), b.cuda(), made(tf, torch, ids, 3), gather=True).cpu()
    assert got[0].isnan().all() and torch.equal(got[1], clean[1]) and torch.equal(got[4:7], clean[4:7])
    assert not got[2:4].isfinite().any() and not got[7].any()


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("how", ["columns", "rows"])
@pytest.mark.parametrize("gather", [False, True])
def test_ragged_gradients(tf, torch, name, shape, how, gather):
    tokens, fan, groups, K, N = shape
    rng = np.random.default_rng(tokens * 5 + N)
    ids = choices(rng, tokens, min(fan, groups), groups)
    fan = ids.shape[1]
    offsets, order, _ = grouping(ids.reshape(-1), groups)
    a = tensor(torch, rng, (tokens if gather else tokens * fan, K), name)
    b, dc = tensor(torch, rng, (groups, K, N), name, K ** -0.5), tensor(torch, rng, (tokens * fan, N), name)
    da, db = tf.ragged_gemm_backward(a.cuda(), layout(torch, b, how), dc.cuda(), made(tf, torch, ids, groups), gather=gather)
    A, B, D = a.double(), b.double(), dc.double()
    want_a, size_a = torch.zeros(A.shape, dtype=torch.float64), torch.zeros(A.shape, dtype=torch.float64)
    parts = torch.zeros(A.shape, dtype=torch.float64)               # the parts that are rounded before they are added up
    want_b, size_b = torch.zeros(B.shape, dtype=torch.float64), torch.zeros(B.shape, dtype=torch.float64)
    for g in range(groups):
        for p in range(offsets[g], offsets[g + 1]):
            s = order[p] // fan if gather else p
            part = D[p] @ B[g].t()
            want_a[s] += part
            parts[s] += part.abs()
            size_a[s] += D[p].abs() @ B[g].abs().t()
            want_b[g] += torch.outer(A[s], D[p])
            size_b[g] += torch.outer(A[s], D[p]).abs()
    extra = HALF_STEP[name] * (1 + 2 ** -6) * parts + fan * SMALLEST[name] if gather and fan > 1 else 0.0
    close(da, want_a, size_a, N + fan, name, extra)
    close(db, want_b, size_b, max(offsets[g + 1] - offsets[g] for g in range(groups)), name)


@pytest.mark.gpu
def test_ragged_weight_gradient_adds_to_what_is_there(tf, torch):
    rng = np.random.default_rng(2)
    ids = choices(rng, 60, 1, 4, only=[0, 2])[:, 0]
    offsets, order, _ = grouping(ids, 4)
    a, dc, db = tensor(torch, rng, (60, 24), "float32"), tensor(torch, rng, (60, 36), "float32"), tensor(torch, rng, (4, 24, 36), "float32")
    want, size = 2.0 * db.double(), 2.0 * db.double().abs()
    for g in range(4):
        rows = torch.tensor(order[offsets[g]:offsets[g + 1]], dtype=torch.long)
        want[g] += 0.25 * a[rows].double().t() @ dc[offsets[g]:offsets[g + 1]].double()
        size[g] += 0.25 * a[rows].double().abs().t() @ dc[offsets[g]:offsets[g + 1]].double().abs()
    out = db.cuda()
    tf.ragged_gemm_grad_into(a.cuda(), dc.cuda(), made(tf, torch, ids, 4), 0.25, 2.0, out, gather=True)
    close(out, want, size, 60, "float32")


@pytest.mark.gpu
def test_ragged_gradients_against_differences(tf, torch):
    rng = np.random.default_rng(4)
    ids = choices(rng, 12, 2, 3)
    g = made(tf, torch, ids, 3)
    a, b, dc = (tensor(torch, rng, s, "float64").cuda() for s in ((12, 9), (3, 9, 7), (24, 7)))
    da, db = tf.ragged_gemm_backward(a, b, dc, g, gather=True)
    for t, grad in ((a, da), (b, db)):
        for _ in range(6):
            d = torch.randn_like(t)
            h = 1e-5      # the product is linear in each operand: the difference has no error but rounding, < 1e-8 here
            value = lambda s: (tf.ragged_gemm(*((t + s * d, b) if t is a else (a, t + s * d)), g, gather=True) * dc).sum()
            assert abs((value(h) - value(-h)) / (2 * h) - (grad * d).sum()) < 1e-8


@pytest.mark.gpu
def test_ragged_product_beyond_32_bit_offsets(tf, torch):
    # the weights, the result and the rows' source each span more than 2^32 bytes
    rng = np.random.default_rng(6)
    groups, K, N = 70, 64, 700000
    b = torch.zeros(groups, K, N, dtype=torch.bfloat16, device="cuda")
    some = tensor(torch, rng, (K, 40), "bfloat16")
    b[69, :, -40:] = some.cuda()
    a = tensor(torch, rng, (3200, K), "bfloat16")
    ids = np.full(3200, 69)
    ids[:5] = 0
    c = tf.ragged_gemm(a.cuda(), b, made(tf, torch, ids, groups), gather=True)
    want, size = a[-6:].double() @ some.double(), a[-6:].double().abs() @ some.double().abs()
    close(c[-6:, -40:], want, size, K, "bfloat16")
    assert not c[:5].any() and not c[-1, :-40].any()
    del b, c
    wide = torch.zeros(3200, 700000, dtype=torch.bfloat16, device="cuda")
    wide[:, -K:] = a.cuda()
    small = tensor(torch, rng, (2, K, 24), "bfloat16")
    c = tf.ragged_gemm(wide[:, -K:], small.cuda(), made(tf, torch, np.ones(3200, int), 2), gather=True)
    close(c, a.double() @ small[1].double(), a.double().abs() @ small[1].double().abs(), K, "bfloat16")


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
def test_ragged_product_of_uneven_groups_of_many_rows(tf, torch, name):
    # groups of 0, 1, 1023 ... rows across many tiles; the reference in blocks
    rng = np.random.default_rng(9)
    counts = [0, 1, 1023, 0, 257, 256, 5, 128, 600, 0, 31]
    ids = np.repeat(np.arange(len(counts)), counts)
    K, N = 320, 288
    offsets = np.cumsum([0] + counts)
    a, b = tensor(torch, rng, (len(ids), K), name), tensor(torch, rng, (len(counts), K, N), name, K ** -0.5)
    for how in ("columns", "rows"):
        g = tf.RowGroups(torch.tensor(offsets, dtype=torch.int32, device="cuda"), n_rows=len(ids))
        got = tf.ragged_gemm(a.cuda(), layout(torch, b, how), g)
        want = torch.cat([a[offsets[i]:offsets[i + 1]].double() @ b[i].double() for i in range(len(counts))])
        size = torch.cat([a[offsets[i]:offsets[i + 1]].double().abs() @ b[i].double().abs() for i in range(len(counts))])
        close(got, want, size, K, name)
        dc = tensor(torch, rng, (len(ids), N), name)
        da, db = tf.ragged_gemm_backward(a.cuda(), layout(torch, b, how), dc.cuda(), g)
        D, A, B = dc.double(), a.double(), b.double()
        cut = [slice(offsets[i], offsets[i + 1]) for i in range(len(counts))]
        close(da, torch.cat([D[s] @ B[i].t() for i, s in enumerate(cut)]), torch.cat([D[s].abs() @ B[i].abs().t() for i, s in enumerate(cut)]), N, name)
        close(db, torch.stack([A[s].t() @ D[s] for s in cut]), torch.stack([A[s].abs().t() @ D[s].abs() for s in cut]), 1023, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("K,N", [(136, 2600), (135, 2599), (20, 12008), (1100, 130)])
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_ragged_product_in_tiles_of_every_size(tf, torch, name, K, N, how):
    # wide results of many rows, short and long sums, rows that start 16-byte aligned and rows that do not; the reference in blocks
    rng = np.random.default_rng(K)
    counts = [0, 1, 1023, 0, 257, 256, 5, 128, 600, 0, 31]
    offsets, rows = np.cumsum([0] + counts), sum(counts)
    a, b, dc = tensor(torch, rng, (rows, K), name), tensor(torch, rng, (len(counts), K, N), name, K ** -0.5), tensor(torch, rng, (rows, N), name)
    g = tf.RowGroups(torch.tensor(offsets, dtype=torch.int32, device="cuda"), n_rows=rows)
    got = tf.ragged_gemm(a.cuda(), layout(torch, b, how), g)
    da, db = tf.ragged_gemm_backward(a.cuda(), layout(torch, b, how), dc.cuda(), g)
    for i, n in enumerate(counts):
        s = slice(offsets[i], offsets[i] + n)
        A, B, D = a[s].cuda().double(), b[i].cuda().double(), dc[s].cuda().double()
        close(got[s], A @ B, A.abs() @ B.abs(), K, name)
        close(da[s], D @ B.t().contiguous(), D.abs() @ B.abs().t().contiguous(), N, name)
        close(db[i], A.t().contiguous() @ D, A.abs().t().contiguous() @ D.abs(), n, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16"])
@pytest.mark.parametrize("K,N", [(128, 2600), (127, 2599)])
def test_ragged_gradient_of_gathered_rows_of_long_groups(tf, torch, name, K, N):
    # several hundred rows of a group, each read by way of the order, some of which lead nowhere
    rng = np.random.default_rng(N)
    tokens, groups = 700, 3
    ids = choices(rng, tokens, 2, groups)
    offsets, order, _ = grouping(ids.reshape(-1), groups)
    gone = rng.choice(offsets[-1], 20, replace=False)
    order = np.asarray(order)
    order[gone[:10]], order[gone[10:]] = -1, 2 * tokens + 5
    a, dc = tensor(torch, rng, (tokens, K), name), tensor(torch, rng, (2 * tokens, N), name)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    db = torch.empty(groups, K, N, dtype=a.dtype, device="cuda")
    tf.ragged_gemm_grad_into(a.cuda(), dc.cuda(), tf.RowGroups(i32(offsets), i32(order), fan=2), 1.0, 0.0, db, gather=True)
    for i in range(groups):
        p = [p for p in range(offsets[i], offsets[i + 1]) if 0 <= order[p] < 2 * tokens]
        A, D = a[order[p] // 2].double(), dc[p].double()
        close(db[i], A.t() @ D, A.abs().t() @ D.abs(), len(p), name)


# ------------------------------------------------------------------------------------------------------ joining
@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,fan,groups,N", [(1, 1, 1, 1), (1, 8, 8, 40), (33, 2, 5, 7), (70, 3, 4, 513), (9, 11, 12, 64), (600, 4, 16, 128)])
@pytest.mark.parametrize("how", ["columns", "pitch", "steps"])
def test_combine_and_its_gradients(tf, torch, name, tokens, fan, groups, N, how):
    rng = np.random.default_rng(tokens + N)
    ids = choices(rng, tokens, fan, groups)
    offsets, order, positions = grouping(ids.reshape(-1), groups)
    wide = torch.float64 if name == "float64" else torch.float32
    x, dy = tensor(torch, rng, (tokens * fan, N), name), tensor(torch, rng, (tokens, N), name)
    w = torch.from_numpy(rng.standard_normal((tokens, fan))).to(wide)
    grouped = np.asarray(positions).reshape(tokens, fan) >= 0
    w[~torch.from_numpy(grouped)] = float("nan")                   # the weight of a choice of no group is never used
    g = made(tf, torch, ids, groups)
    y = tf.combine_rows(layout(torch, x, how), g, w.cuda())
    dx, dw = tf.combine_rows_backward(layout(torch, x, how), layout(torch, w, "steps"), layout(torch, dy, how), g)
    plain = tf.combine_rows(x.cuda(), g)
    X, D, W = x.double(), dy.double(), w.double()
    want, size, ones, ones_size = (torch.zeros(tokens, N, dtype=torch.float64) for _ in range(4))
    want_x = torch.zeros(tokens * fan, N, dtype=torch.float64)
    want_w, size_w = torch.zeros(tokens, fan, dtype=torch.float64), torch.zeros(tokens, fan, dtype=torch.float64)
    for t, j in itertools.product(range(tokens), range(fan)):
        p = positions[t * fan + j]
        if p < 0:
            continue
        want[t] += W[t, j] * X[p]
        size[t] += (W[t, j] * X[p]).abs()
        ones[t] += X[p]
        ones_size[t] += X[p].abs()
        want_x[p] = W[t, j] * D[t]
        want_w[t, j], size_w[t, j] = X[p] @ D[t], X[p].abs() @ D[t].abs()
    close(y, want, size, fan, name)
    close(plain, ones, ones_size, fan, name)
    close(dx, want_x, want_x.abs(), 1, name)
    close(dw, want_w, size_w, N, "float64" if name == "float64" else "float32")
    only_x, none = tf.combine_rows_backward(x.cuda(), None, dy.cuda(), g)
    assert none is None
    close(only_x, torch.where(torch.tensor([p in set(positions) for p in range(tokens * fan)])[:, None], D[torch.tensor(order) // fan], 0.0), D.abs().max() * torch.ones(1), 1, name)


# ------------------------------------------------------------------------------------------------------ adapters
def adapter_reference(torch, x, w, a, b, scales, ids):
    X, W, A, B = x.double(), w.double(), a.double(), b.double()
    y, size, low = X @ W, X.abs() @ W.abs(), torch.zeros(X.shape[0], W.shape[1], dtype=torch.float64)
    for t, g in enumerate(ids):
        if 0 <= g < A.shape[0]:
            s = 1.0 if scales is None else float(scales[g])
            y[t] += s * (X[t] @ A[g] @ B[g])
            low[t] = abs(s) * (X[t].abs() @ A[g].abs() @ B[g].abs())
    return y, size + low, low


ADAPTERS = [(1, 1, 1, 1, 1), (1, 3, 64, 40, 4), (5, 2, 33, 17, 7), (64, 32, 136, 200, 16), (100, 3, 72, 65, 24), (200, 4, 256, 130, 50), (130, 64, 96, 128, 100), (20, 2, 64, 64, 200),
            (900, 3, 128, 320, 32), (700, 2, 192, 264, 64), (300, 5, 72, 136, 128), (450, 1, 64, 256, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,groups,K,N,R", ADAPTERS)
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_adapters_and_their_gradients(tf, torch, name, tokens, groups, K, N, R, how):
    rng = np.random.default_rng(tokens + K + R)
    ids = choices(rng, tokens, 1, groups, none=0.25)[:, 0]
    wide = torch.float64 if name == "float64" else torch.float32
    x, w = tensor(torch, rng, (tokens, K), name), tensor(torch, rng, (K, N), name, K ** -0.5)
    a, b = tensor(torch, rng, (groups, K, R), name, K ** -0.5), tensor(torch, rng, (groups, R, N), name, R ** -0.5)
    scales = torch.from_numpy(0.2 + rng.random(groups)).to(wide)
    dy = tensor(torch, rng, (tokens, N), name)
    g = made(tf, torch, ids, groups)
    on = [layout(torch, t, how) for t in (w, a, b)]
    want, size, low = adapter_reference(torch, x, w, a, b, scales, ids)
    close(tf.adapter_gemm(x.cuda(), *on, g, scales.cuda()), want, size, K + R, name, MIDDLE[name] * low)
    want, size, low = adapter_reference(torch, x, w, a, b, None, ids)
    close(tf.adapter_gemm(x.cuda(), *on, g), want, size, K + R, name, MIDDLE[name] * low)
    dx, da, db = tf.adapter_gemm_backward(x.cuda(), *on, dy.cuda(), g, scales.cuda())
    want, size, low = adapter_reference(torch, dy, w.t(), b.transpose(1, 2), a.transpose(1, 2), scales, ids)
    close(dx, want, size, N + R, name, MIDDLE[name] * low)
    X, D, A, B, S = x.double(), dy.double(), a.double(), b.double(), scales.double()
    for i in range(groups):
        rows = torch.tensor(np.nonzero(ids == i)[0])
        xg, dg = X[rows], D[rows]
        u, ua = dg @ B[i].t(), dg.abs() @ B[i].abs().t()
        v, va = xg @ A[i], xg.abs() @ A[i].abs()
        size = S[i] * xg.abs().t() @ ua
        close(da[i], S[i] * xg.t() @ u, size, len(rows) + N, name, MIDDLE[name] * size)
        size = S[i] * va.t() @ dg.abs()
        close(db[i], S[i] * v.t() @ dg, size, len(rows) + K, name, MIDDLE[name] * size)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16", "float32"])
def test_an_adapter_that_is_no_number_stays_with_its_rows(tf, torch, name):
    rng = np.random.default_rng(1)
    ids = np.array([0, 1, 2, -1, 1, 0, 2, 9])
    x, w = tensor(torch, rng, (8, 64), name), tensor(torch, rng, (64, 48), name, 0.125)
    a, b = tensor(torch, rng, (3, 64, 8), name, 0.125), tensor(torch, rng, (3, 8, 48), name)
    g = made(tf, torch, ids, 3)
    clean = tf.adapter_gemm(x.cuda(), w.cuda(), a.cuda(), b.cuda(), g).cpu()
    b[1], a[2, 5, 3] = float("inf"), float("nan")
    got = tf.adapter_gemm(x.cuda(), w.cuda(), a.cuda(), b.cuda(), g).cpu()
    for t in (0, 3, 5, 7):
        assert torch.equal(got[t], clean[t])
    for t in (1, 2, 4, 6):
        assert not got[t].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("K,N,R", [(72, 6104, 24), (71, 6101, 7), (264, 328, 16)])
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_adapters_of_many_rows_keep_what_is_no_number(tf, torch, name, K, N, R, how):
    # tiles of every size; one adapter infinite, one partly no number, rows of none between them: the others' rows are as they
    # should be, theirs are no numbers
    rng = np.random.default_rng(N)
    ids = np.repeat([2, -1, 0, 1, 3, 0], [260, 7, 300, 5, 290, 130])
    x, w = tensor(torch, rng, (len(ids), K), name), tensor(torch, rng, (K, N), name, K ** -0.5)
    a, b = tensor(torch, rng, (4, K, R), name, K ** -0.5), tensor(torch, rng, (4, R, N), name)
    broken_a, broken_b = a.clone(), b.clone()
    broken_b[1], broken_a[3, K // 2, R - 1] = float("inf"), float("nan")
    got = tf.adapter_gemm(x.cuda(), layout(torch, w, how), layout(torch, broken_a, how), layout(torch, broken_b, how), made(tf, torch, ids, 4)).cpu()
    want, size, low = adapter_reference(torch, x, w, a, b, None, ids)
    kept = torch.from_numpy((ids != 1) & (ids != 3))
    close(got[kept], want[kept], size[kept], K + R, name, MIDDLE[name] * low[kept])
    assert not got[~kept].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("name,big", [("float16", 3.0e4), ("bfloat16", 1.0e30), ("float32", 1.0e30)])
def test_an_adapters_middle_may_exceed_the_operands_range(tf, torch, name, big):
    # x a is 64 * big (beyond f16's largest 65504), x a b again in range
    x = torch.full((6, 64), 1.0, dtype=getattr(torch, name))
    a, b = torch.full((2, 64, 4), big, dtype=x.dtype), torch.full((2, 4, 24), 2.0 ** -13 if name == "float16" else 2.0 ** -60, dtype=x.dtype)
    w = torch.zeros(64, 24, dtype=x.dtype)
    ids = np.array([0, 1, 0, 1, -1, 0])
    want, size, low = adapter_reference(torch, x, w, a, b, None, ids)
    assert want.abs().max() < 6e4 or name != "float16"
    close(tf.adapter_gemm(x.cuda(), w.cuda(), a.cuda(), b.cuda(), made(tf, torch, ids, 2)), want, size, 68, name, MIDDLE[name] * low)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float32", "float64"])
@pytest.mark.parametrize("K,N", [(64, 48), (37, 21), (600, 72)])
def test_products_of_views_with_negative_and_zero_strides(tf, torch, name, K, N):
    rng = np.random.default_rng(K)
    rows, groups, size = 70, 3, torch.finfo(getattr(torch, name)).bits // 8
    code = {"bfloat16": tf.BF16, "float32": tf.F32, "float64": tf.F64}[name]
    a, b = tensor(torch, rng, (rows, K), name), tensor(torch, rng, (groups, K, N), name, K ** -0.5)
    A, B = a.cuda(), b.cuda()
    g = tf.RowGroups(torch.tensor([0, 30, 31, 64], dtype=torch.int32, device="cuda"), n_rows=rows)
    at = lambda t, dims, strides, first: view(tf, dims, strides, t.data_ptr() + first * size)
    stream = torch.cuda.current_stream().cuda_stream

    def run(va, vb, a, b):
        c = torch.zeros(rows, N, dtype=A.dtype, device="cuda")
        vc = at(c, [rows, N], [-N, 1], (rows - 1) * N)          # its rows backwards
        tf._check(tf.lib().tfh_ragged_gemm(code, C.byref(g._c), 4, 1.0, va, vb, 0.0, vc, stream))
        want, size_of = ragged_reference(torch, a, b, [0, 30, 31, 64], list(range(rows)), 1, False)
        close(c.flip(0), want, size_of, K, name)

    plain_a, plain_b = at(A, [rows, K], [K, 1], 0), at(B, [groups, K, N], [K * N, N, 1], 0)
    run(at(A, [rows, K], [-K, 1], (rows - 1) * K), plain_b, a.flip(0), b)
    run(at(A, [rows, K], [0, 1], 5 * K), plain_b, a[5].expand(rows, K), b)
    run(at(A, [rows, K], [K, -1], K - 1), plain_b, a.flip(1), b)
    run(plain_a, at(B, [groups, K, N], [-K * N, N, 1], (groups - 1) * K * N), a, b.flip(0))
    run(plain_a, at(B, [groups, K, N], [K * N, -N, 1], (K - 1) * N), a, b.flip(1))
    run(plain_a, at(B, [groups, K, N], [0, N, 1], K * N), a, b[1].expand(groups, K, N))
    run(plain_a, at(B, [groups, K, N], [K * N, 0, 1], 0), a, b[:, :1].expand(groups, K, N))
    db = torch.zeros(groups, K, N, dtype=A.dtype, device="cuda")
    dc = tensor(torch, rng, (rows, N), name)
    D = dc.cuda()
    tf._check(tf.lib().tfh_ragged_gemm_grad(code, C.byref(g._c), 0, 1.0, at(A, [rows, K], [-K, 1], (rows - 1) * K), at(D, [rows, N], [-N, 1], (rows - 1) * N), 0.0,
                                            at(db, [groups, K, N], [K * N, -N, 1], (K - 1) * N), stream))
    for i, (x, y) in enumerate([(0, 30), (30, 31), (31, 64)]):
        X, Y = a.flip(0)[x:y].double(), dc.flip(0)[x:y].double()
        close(db[i].flip(0), X.t() @ Y, X.abs().t() @ Y.abs(), y - x, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("K,N,R", [(96, 160, 16), (35, 17, 5)])
def test_adapters_of_rows_that_lie_in_order(tf, torch, name, K, N, R):
    # no order: the groups' rows one after the other, the last ones of none
    rng = np.random.default_rng(R)
    ids = np.repeat([0, 1, 2, -1], [40, 1, 70, 6])
    x, w = tensor(torch, rng, (len(ids), K), name), tensor(torch, rng, (K, N), name, K ** -0.5)
    a, b, dy = tensor(torch, rng, (3, K, R), name, K ** -0.5), tensor(torch, rng, (3, R, N), name), tensor(torch, rng, (len(ids), N), name)
    g = tf.RowGroups(torch.tensor([0, 40, 41, 111], dtype=torch.int32, device="cuda"), n_rows=len(ids))
    want, size, low = adapter_reference(torch, x, w, a, b, None, ids)
    close(tf.adapter_gemm(x.cuda(), w.cuda(), a.cuda(), b.cuda(), g), want, size, K + R, name, MIDDLE[name] * low)
    listed = made(tf, torch, ids, 3)
    one, other = (tf.adapter_gemm_backward(x.cuda(), w.cuda(), a.cuda(), b.cuda(), dy.cuda(), h) for h in (g, listed))
    assert all(torch.equal(p, q) for p, q in zip(one, other))


# ------------------------------------------------------------------------------------------------------ together, streams, graphs
def expert_layer(tf, x, up, down, ids, gates):
    groups = tf.RowGroups.from_ids(ids, up.shape[0])
    h = tf.ragged_gemm(x, up, groups, gather=True)
    return tf.combine_rows(tf.ragged_gemm(h, down, groups), groups, gates), groups, h


def expert_gradients(tf, x, up, down, gates, dy, groups, h):
    z = tf.ragged_gemm(h, down, groups)
    dz, dgates = tf.combine_rows_backward(z, gates, dy, groups)
    dh, ddown = tf.ragged_gemm_backward(h, down, dz, groups)
    dx, dup = tf.ragged_gemm_backward(x, up, dh, groups, gather=True)
    return dx, dup, ddown, dgates


def layer_inputs(torch, seed, name="float32", tokens=48, fan=2, groups=6, K=40, N=56):
    rng = np.random.default_rng(seed)
    x, up, down = tensor(torch, rng, (tokens, K), name), tensor(torch, rng, (groups, K, N), name, K ** -0.5), tensor(torch, rng, (groups, N, K), name, N ** -0.5)
    ids = torch.from_numpy(choices(rng, tokens, fan, groups))
    gates = torch.softmax(torch.from_numpy(rng.standard_normal((tokens, fan))), 1).to(torch.float64 if name == "float64" else torch.float32)
    return [t.cuda() for t in (x, up, down, ids, gates, tensor(torch, rng, (tokens, K), name))]


@pytest.mark.gpu
def test_a_layer_of_experts_and_its_gradients_together(tf, torch):
    x, up, down, ids, gates, dy = layer_inputs(torch, 0, "float64")
    y, groups, h = expert_layer(tf, x, up, down, ids, gates)
    got = expert_gradients(tf, x, up, down, gates, dy, groups, h)
    leaves = [t.cpu().clone().requires_grad_() for t in (x, up, down, gates)]
    X, UP, DOWN, GATES = leaves
    rows = []
    for t in range(X.shape[0]):
        total = torch.zeros(X.shape[1], dtype=torch.float64)
        for j, e in enumerate(ids[t].tolist()):
            if 0 <= e < UP.shape[0]:
                total = total + GATES[t, j] * (X[t] @ UP[e] @ DOWN[e])
        rows.append(total)
    Y = torch.stack(rows)
    want = torch.autograd.grad((Y * dy.cpu()).sum(), leaves)
    assert (y.cpu() - Y).abs().max() < 1e-12          # sums of 40, 56 and 2 products of order one in 64 bits
    for a, b in zip((got[0], got[1], got[2], got[3]), want):
        assert (a.cpu() - b).abs().max() < 1e-11


@pytest.mark.gpu
def test_calls_on_another_stream_and_on_tensors(tf, torch):
    x, up, down, ids, gates, dy = layer_inputs(torch, 1)
    want, _, _ = expert_layer(tf, x, up, down, ids, gates)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    st = side.cuda_stream
    groups = tf.RowGroups.from_ids(ids, up.shape[0], stream=st)
    h = tf.ragged_gemm(x, up, groups, gather=True, stream=st)
    y = tf.combine_rows(tf.ragged_gemm(h, down, groups, stream=st), groups, gates, stream=st)
    del h
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    T = tf.Tensor.from_torch
    groups = tf.RowGroups.from_ids(ids, up.shape[0], stream=st)      # its event orders the current stream's calls behind it
    out = tf.combine_rows(tf.ragged_gemm(tf.ragged_gemm(T(x), T(up), groups, gather=True), T(down), groups), groups, T(gates))
    assert isinstance(out, tf.Tensor) and out.event is not None
    assert np.array_equal(out.to_numpy(), want.cpu().numpy())
    assert tf.Tensor.from_torch(x.bfloat16()).to_numpy().dtype == np.float32


@pytest.mark.gpu
def test_two_streams_at_once(tf, torch):
    # the same operands on two streams, nothing waited for in between: workspaces of their own
    x, up, down, ids, gates, dy = layer_inputs(torch, 11, "bfloat16", tokens=2000, fan=2, groups=5, K=136, N=264)
    low_a, low_b = up[:, :, :8].contiguous(), up[:, :8, :].contiguous()
    flat = tf.RowGroups.from_ids(ids[:, 0], up.shape[0])
    want = (expert_layer(tf, x, up, down, ids, gates)[0], tf.adapter_gemm(x, up[0].contiguous(), low_a, low_b, flat))
    torch.cuda.synchronize()
    out = []
    for side in [torch.cuda.Stream() for _ in range(2)] * 3:
        with torch.cuda.stream(side):
            out.append((expert_layer(tf, x, up, down, ids, gates)[0], tf.adapter_gemm(x, up[0].contiguous(), low_a, low_b, flat)))
    torch.cuda.synchronize()
    for got in out:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float32"])
def test_captured_calls_replay_on_new_choices(tf, torch, name):
    x, up, down, ids, gates, dy = layer_inputs(torch, 2, name)
    others = [layer_inputs(torch, s, name) for s in (3, 4, 5)]
    low_a, low_b = up[:, :, :8].contiguous(), up[:, :8, :].contiguous()
    weights = up[0].contiguous()

    def everything():
        y, groups, h = expert_layer(tf, x, up, down, ids, gates)
        flat = tf.RowGroups.from_ids(ids[:, 0], up.shape[0])
        z = tf.adapter_gemm(x, weights, low_a, low_b, flat)
        return (y, z) + expert_gradients(tf, x, up, down, gates, dy, groups, h) + tf.adapter_gemm_backward(x, weights, low_a, low_b, z, flat)

    everything()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                       # two graphs, each with buffers of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = everything()
        graphs.append((graph, out))
    for new in others:
        for t, n in zip((x, ids, gates, dy), (new[0], new[3], new[4], new[5])):
            t.copy_(n)
        want = [t.clone() for t in everything()]
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits(tf, torch):
    x, up, down, ids, gates, dy = layer_inputs(torch, 7, "bfloat16", tokens=300, fan=3, groups=5, K=136, N=264)
    first = None
    for _ in range(3):
        y, groups, h = expert_layer(tf, x, up, down, ids, gates)
        out = (y,) + expert_gradients(tf, x, up, down, gates, dy, groups, h)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


@pytest.mark.gpu
def test_lists_that_lead_nowhere_stay_inside_the_views(tf, torch):
    # offsets, orders and positions beyond the rows are treated as absent
    a = torch.ones(8, 16, dtype=torch.bfloat16, device="cuda")
    b = torch.ones(3, 16, 8, dtype=torch.bfloat16, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    g = tf.RowGroups(i32([0, 3, 900, 1000]), i32([0, 1, 77, -3, 4, 5, 2000000000, 7]), i32([0, 900, -7, 3, 4, 5, 6, 7]))
    c = tf.ragged_gemm(a, b, g, gather=True).cpu()
    assert [float(v) for v in c[:, 0]] == [16, 16, 0, 0, 16, 16, 0, 16]
    y = tf.combine_rows(a, g).cpu()
    assert [float(v) for v in y[:, 0]] == [1, 0, 0, 1, 1, 1, 1, 1]
    g = tf.RowGroups(i32([-5, 6, 2, 8]), n_rows=8)                 # not ascending: the middle group has no rows
    tf.ragged_gemm(a, b, g)
    tf.adapter_gemm(a, b[0], b, torch.ones(3, 8, 8, dtype=torch.bfloat16, device="cuda"), g)
    tf.ragged_gemm_backward(a, b, torch.ones(8, 8, dtype=torch.bfloat16, device="cuda"), g)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------------ refusals (no GPU)
def view(tf, dims, strides=None, base=4096, flags=0):
    v = tf.tfh_view()
    v.base, v.rank, v.flags, v.offset = base, len(dims), flags, 0
    if strides is None:
        strides = [int(np.prod(dims[i + 1:])) for i in range(len(dims))]
    for i, (d, s) in enumerate(zip(dims, strides)):
        v.dims[i], v.strides[i] = d, s
    return C.byref(v)


def row_groups(tf, n_rows=8, n_groups=3, fan=1, offsets=4096, order=4096, positions=4096):
    from tenferro_rs_amd.row_groups import tfh_row_groups
    return C.byref(tfh_row_groups(offsets, order, positions, n_rows, n_groups, fan))


def refused(tf, call, error):
    with pytest.raises(error) as e:
        tf._check(call)
    return e.value


def test_products_refuse_what_does_not_fit(tf):
    L, V, G = tf.lib(), lambda *d, **k: view(tf, d, **k), lambda **k: row_groups(tf, **k)
    run = lambda dt=4, g=None, fl=0, a=None, b=None, c=None: L.tfh_ragged_gemm(dt, g or G(), fl, 1.0, a or V(8, 16), b or V(3, 16, 24), 0.0, c or V(8, 24), None)
    for dt in (2, 3, -1, 6):
        refused(tf, run(dt=dt), tf.InvalidArgument)
    e = refused(tf, run(a=V(7, 16)), tf.ShapeMismatch)
    assert e.expected == [8, 16] and e.got == [7, 16]
    refused(tf, run(a=V(8, 16, 1)), tf.RankMismatch)
    refused(tf, run(b=V(16, 24)), tf.RankMismatch)
    assert refused(tf, run(b=V(3, 17, 24)), tf.ShapeMismatch).expected == [3, 16, 24]
    refused(tf, run(b=V(4, 16, 24)), tf.ShapeMismatch)
    refused(tf, run(c=V(8, 25)), tf.ShapeMismatch)
    refused(tf, run(c=V(8, 24, strides=[0, 1])), tf.InvalidArgument)
    refused(tf, run(a=V(8, 16, base=0)), tf.InvalidArgument)
    refused(tf, run(a=V(8, 16, flags=1)), tf.InvalidArgument)
    refused(tf, run(fl=8), tf.InvalidArgument)
    refused(tf, run(fl=1, g=G(order=None)), tf.InvalidArgument)
    refused(tf, run(fl=2, g=G(order=None)), tf.InvalidArgument)
    refused(tf, run(fl=1, g=G(fan=2)), tf.ShapeMismatch)               # gathered: A has n_rows / fan rows
    for bad in (dict(n_groups=0), dict(n_rows=-1), dict(fan=0), dict(fan=3), dict(offsets=None), dict(n_rows=1 << 40)):
        refused(tf, run(g=G(**bad)), tf.InvalidArgument)
    refused(tf, L.tfh_ragged_gemm(4, None, 0, 1.0, V(8, 16), V(3, 16, 24), 0.0, V(8, 24), None), tf.InvalidArgument)
    refused(tf, L.tfh_ragged_gemm(4, G(), 0, 1.0, None, V(3, 16, 24), 0.0, V(8, 24), None), tf.InvalidArgument)
    grad = lambda fl=0, a=None, dc=None, db=None: L.tfh_ragged_gemm_grad(4, G(), fl, 1.0, a or V(8, 16), dc or V(8, 24), 0.0, db or V(3, 16, 24), None)
    refused(tf, grad(fl=4), tf.InvalidArgument)
    refused(tf, grad(dc=V(9, 24)), tf.ShapeMismatch)
    refused(tf, grad(db=V(3, 24, 16)), tf.ShapeMismatch)


@pytest.mark.parametrize("big", [0x7ff00001, 0x7fffffff, 1 << 31, 1 << 40])
def test_what_32_bit_indices_cannot_walk_is_refused(tf, big):
    L, V, G = tf.lib(), lambda *d: view(tf, d), lambda **k: row_groups(tf, **k)
    refused(tf, L.tfh_ragged_gemm(4, G(n_rows=1), 0, 1.0, V(1, 16), V(3, 16, big), 0.0, V(1, big), None), tf.InvalidArgument)
    refused(tf, L.tfh_ragged_gemm(4, G(n_rows=1), 0, 1.0, V(1, big), V(3, big, 16), 0.0, V(1, 16), None), tf.InvalidArgument)
    refused(tf, L.tfh_ragged_gemm(4, G(n_rows=big), 0, 1.0, V(big, 16), V(3, 16, 16), 0.0, V(big, 16), None), tf.InvalidArgument)
    refused(tf, L.tfh_ragged_gemm_grad(4, G(n_rows=1), 0, 1.0, V(1, big), V(1, 8), 0.0, V(3, big, 8), None), tf.InvalidArgument)
    refused(tf, L.tfh_combine_rows(4, G(n_rows=1), V(1, big), None, V(1, big), None), tf.InvalidArgument)
    refused(tf, L.tfh_group_rows(32, V(big), 4, 4096, 4096, None, 4096, 1 << 40, None), tf.InvalidArgument)
    if big <= 0x7fffffff:
        refused(tf, L.tfh_ragged_gemm(4, G(n_groups=big), 0, 1.0, V(8, 16), V(big, 16, 8), 0.0, V(8, 8), None), tf.InvalidArgument)


def test_grouping_refuses_what_does_not_fit(tf):
    L = tf.lib()
    run = lambda bits=32, ids=None, n=4, off=4096, order=4096, ws=4096, b=1 << 20: L.tfh_group_rows(bits, ids or view(tf, [8]), n, off, order, None, ws, b, None)
    refused(tf, run(bits=16), tf.InvalidArgument)
    refused(tf, run(n=0), tf.InvalidArgument)
    refused(tf, run(n=2049), tf.InvalidArgument)
    refused(tf, run(ids=view(tf, [2, 2, 2])), tf.RankMismatch)
    refused(tf, run(ids=view(tf, [8], base=0)), tf.InvalidArgument)
    refused(tf, run(ids=view(tf, [1 << 20, 1 << 20])), tf.InvalidArgument)
    refused(tf, run(off=None), tf.InvalidArgument)
    refused(tf, run(order=None), tf.InvalidArgument)
    refused(tf, run(ids=view(tf, [100000]), b=16), tf.InvalidArgument)
    refused(tf, run(ids=view(tf, [100000]), ws=4100), tf.InvalidArgument)
    assert L.tfh_group_rows_workspace(100, 4) == 0 and L.tfh_group_rows_workspace(1 << 20, 4) > 0


def test_joining_refuses_what_does_not_fit(tf):
    L, V, G = tf.lib(), lambda *d, **k: view(tf, d, **k), lambda **k: row_groups(tf, **dict(dict(fan=2), **k))
    run = lambda g=None, x=None, w=None, y=None: L.tfh_combine_rows(4, g or G(), x or V(8, 6), w, y or V(4, 6), None)
    refused(tf, run(g=G(positions=None)), tf.InvalidArgument)
    refused(tf, run(x=V(8, 7)), tf.ShapeMismatch)
    refused(tf, run(y=V(8, 6)), tf.ShapeMismatch)
    refused(tf, run(w=V(2, 4)), tf.ShapeMismatch)
    refused(tf, run(y=V(4)), tf.RankMismatch)
    refused(tf, L.tfh_combine_rows_grad(4, G(), V(8, 6), None, V(4, 6), V(8, 5), None, None), tf.ShapeMismatch)
    refused(tf, L.tfh_combine_rows_grad(4, G(), None, None, V(4, 6), V(8, 6), V(4, 2), None), tf.InvalidArgument)


def test_adapters_refuse_what_does_not_fit(tf):
    L, V, G = tf.lib(), lambda *d, **k: view(tf, d, **k), lambda **k: row_groups(tf, **k)
    ok = dict(x=V(8, 16), w=V(16, 24), a=V(3, 16, 4), b=V(3, 4, 24), s=None, y=V(8, 24))

    def run(g=None, ws=4096, nb=1 << 20, **k):
        v = dict(ok, **k)
        return L.tfh_adapter_gemm(4, g or G(), v["x"], v["w"], v["a"], v["b"], v["s"], v["y"], ws, nb, None)

    refused(tf, run(g=G(fan=2)), tf.InvalidArgument)
    refused(tf, run(x=V(8, 15)), tf.ShapeMismatch)
    refused(tf, run(a=V(3, 16)), tf.RankMismatch)
    refused(tf, run(b=V(3, 5, 24)), tf.ShapeMismatch)
    refused(tf, run(b=V(2, 4, 24)), tf.ShapeMismatch)
    refused(tf, run(y=V(8, 16)), tf.ShapeMismatch)
    refused(tf, run(s=V(4)), tf.ShapeMismatch)
    refused(tf, run(s=V(3, strides=[2])), tf.Strided)
    refused(tf, run(ws=None), tf.InvalidArgument)
    refused(tf, run(nb=L.tfh_adapter_workspace(4, 8, 4, 0) - 1), tf.InvalidArgument)
    refused(tf, run(ws=4104), tf.InvalidArgument)
    assert L.tfh_adapter_workspace(4, 8, 4, 1) > L.tfh_adapter_workspace(4, 8, 4, 0) >= 8 * 4 * 4 and L.tfh_adapter_workspace(4, 8, 0, 1) == 0
    refused(tf, L.tfh_adapter_gemm_grad(4, G(), ok["x"], ok["w"], ok["a"], ok["b"], None, V(8, 24), None, V(3, 16, 5), None, 4096, 1 << 20, None), tf.ShapeMismatch)


def test_what_has_no_place_on_the_gpu_is_refused_by_name(tf):
    import torch
    with pytest.raises(tf.NoCompatibleComputeDevice):
        tf.RowGroups.from_ids(torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(tf.NoCompatibleComputeDevice):
        tf.RowGroups(torch.zeros(3, dtype=torch.int32), n_rows=4)
    with pytest.raises(tf.InvalidArgument):
        tf.ragged_gemm(torch.zeros(4, 4), torch.zeros(1, 4, 4), None)


@pytest.mark.parametrize("call", ["plan", "fill", "conj"])
def test_16_bit_types_are_refused_elsewhere(tf, call):
    L = tf.lib()
    for dt in (tf.BF16, tf.F16):
        assert L.tfh_dtype_size(dt) == 2
        if call == "plan":
            with pytest.raises(tf.InvalidArgument):
                tf.HipBackend.plan(dt, tf.PrimDescriptor.Contract([0, 1], [1, 2], [0, 2]), [[2, 3], [3, 4], [2, 4]])
            assert not tf.HipBackend.has_extension_for(dt, tf.Extension.Contract)
        elif call == "fill":
            refused(tf, L.tfh_fill(dt, (C.c_double * 2)(), view(tf, [4]), None), tf.InvalidArgument)
        else:
            refused(tf, L.tfh_conj(dt, view(tf, [4]), view(tf, [4]), None), tf.InvalidArgument)


# ------------------------------------------------------------------------------------------------------ sums that are rounded once
def rows_gradient_reference(torch, dc, b, offsets, order, fan):
    """The gradient of the gathered rows in 64 bits and the sums of absolute values."""
    D, B = dc.double(), b.double()
    want, size = (torch.zeros(len(order) // fan, B.shape[1], dtype=torch.float64) for _ in range(2))
    for g in range(len(offsets) - 1):
        p = slice(offsets[g], offsets[g + 1])
        s = torch.tensor([o // fan for o in order[p]], dtype=torch.long)
        want.index_add_(0, s, D[p] @ B[g].t())
        size.index_add_(0, s, D[p].abs() @ B[g].abs().t())
    return want, size


GRADIENT_SHAPES = [  # tokens, fan, groups, K, N: few rows, tiles of every size, k shared out, rows that start at any address
    (1, 2, 2, 1, 1), (9, 3, 5, 33, 5), (24, 2, 4, 264, 128), (70, 8, 9, 65, 129), (300, 2, 3, 136, 72), (900, 3, 4, 2048, 264), (900, 3, 4, 4104, 128), (700, 2, 2, 2047, 135)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", GRADIENT_SHAPES, ids=str)
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_the_gradient_of_gathered_rows_is_rounded_once(tf, torch, name, shape, how):
    # no slack for a rounding of each choice's part: the sum of the parts in 32 bits, as any other
    tokens, fan, groups, K, N = shape
    rng = np.random.default_rng(tokens + K)
    ids = choices(rng, tokens, fan, groups)
    offsets, order, _ = grouping(ids.reshape(-1), groups)
    a, b, dc = tensor(torch, rng, (tokens, K), name), tensor(torch, rng, (groups, K, N), name, N ** -0.5), tensor(torch, rng, (tokens * fan, N), name)
    want, size = rows_gradient_reference(torch, dc, b, offsets, order, fan)
    da, _ = tf.ragged_gemm_backward(a.cuda(), layout(torch, b, how), dc.cuda(), made(tf, torch, ids, groups), gather=True)
    close(da, want, size, N + fan, name)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,K,N", [(3, 5, 7), (20, 72, 64), (300, 136, 72), (1200, 2048, 264)])
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_parts_of_a_gradient_beyond_the_range_may_cancel(tf, torch, tokens, K, N, how):
    # two choices of a token, of opposite sign: the parts are (N - 1) 2^22 and 2^11 more, beyond f16's largest, 65504, their sum is 2^11.
    # All are whole multiples of 2^11 below 2^(11 + 24): exact in 32 bits, in any order.
    big = 2.0 ** 11
    ids = np.stack([np.arange(tokens) % 2, 1 - np.arange(tokens) % 2], 1)
    b, dc = torch.full((2, K, N), big, dtype=torch.float16), torch.full((2 * tokens, N), big, dtype=torch.float16)
    b[1], b[1, :, N - 1] = -big, 0
    dc[:, N - 1] = 1
    da, _ = tf.ragged_gemm_backward(torch.zeros(tokens, K, dtype=torch.float16, device="cuda"), layout(torch, b, how), dc.cuda(), made(tf, torch, ids, 2), gather=True)
    assert torch.equal(da.cpu(), torch.full((tokens, K), big, dtype=torch.float16))


@pytest.mark.gpu
def test_the_rows_gradient_by_its_own_entry(tf, torch):
    # alpha, strides of its operands and its result, rows of no group: zeros
    rng = np.random.default_rng(21)
    tokens, fan, groups, K, N = 60, 2, 3, 40, 24
    ids = choices(rng, tokens, fan, groups, none=0.4)
    offsets, order, _ = grouping(ids.reshape(-1), groups)
    b, dc = tensor(torch, rng, (groups, K, N), "bfloat16"), tensor(torch, rng, (tokens * fan, N), "bfloat16")
    g = made(tf, torch, ids, groups)
    want, size = rows_gradient_reference(torch, dc, b, offsets, order, fan)
    L, at = tf.lib(), lambda t: view(tf, list(t.shape), list(t.stride()), t.data_ptr())
    need = L.tfh_ragged_gemm_grad_a_workspace(tf.BF16, tokens * fan, K, fan, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for how in ("columns", "rows", "pitch", "steps"):
        out = layout(torch, torch.full((tokens, K), float("nan"), dtype=torch.bfloat16), how)
        B, D = layout(torch, b, how), layout(torch, dc, how)
        tf._check(L.tfh_ragged_gemm_grad_a(tf.BF16, C.byref(g._c), 1, -0.5, at(D), at(B), at(out), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
        close(out, -0.5 * want, 0.5 * size, N + fan, "bfloat16")
        gone = torch.from_numpy(((ids < 0) | (ids >= groups)).all(1))
        assert gone.any() and not out.cpu()[gone].any()


def test_the_rows_gradient_refuses_what_does_not_fit(tf):
    L, V, G = tf.lib(), lambda *d, **k: view(tf, d, **k), lambda **k: row_groups(tf, **dict(dict(fan=2), **k))

    def run(dt=4, g=None, fl=1, dc=None, b=None, da=None, ws=4096, nb=1 << 20):
        return L.tfh_ragged_gemm_grad_a(dt, g or G(), fl, 1.0, dc or V(8, 24), b or V(3, 16, 24), da or V(4, 16), ws, nb, None)

    refused(tf, run(dt=3), tf.InvalidArgument)
    refused(tf, run(fl=2), tf.InvalidArgument)
    refused(tf, run(g=G(order=None)), tf.InvalidArgument)
    refused(tf, run(g=G(positions=None)), tf.InvalidArgument)
    refused(tf, L.tfh_ragged_gemm_grad_a(4, None, 1, 1.0, V(8, 24), V(3, 16, 24), V(4, 16), 4096, 1 << 20, None), tf.InvalidArgument)
    refused(tf, run(dc=V(7, 24)), tf.ShapeMismatch)
    refused(tf, run(dc=V(8, 24, 1)), tf.RankMismatch)
    refused(tf, run(b=V(3, 16, 25)), tf.ShapeMismatch)
    refused(tf, run(da=V(8, 16)), tf.ShapeMismatch)
    refused(tf, run(fl=0), tf.ShapeMismatch)
    refused(tf, run(da=V(4, 16, strides=[0, 1])), tf.InvalidArgument)
    refused(tf, run(ws=None), tf.InvalidArgument)
    refused(tf, run(ws=4104), tf.InvalidArgument)
    need = L.tfh_ragged_gemm_grad_a_workspace(4, 8, 16, 2, 1)
    assert need == 8 * 16 * 4
    refused(tf, run(nb=need - 1), tf.InvalidArgument)
    assert L.tfh_ragged_gemm_grad_a_workspace(4, 8, 16, 2, 0) == 0 and L.tfh_ragged_gemm_grad_a_workspace(4, 8, 16, 1, 1) == 0


# ------------------------------------------------------------------------------------------------------ infinities of the adapters' operands
def agree(got, want, size, k, name, extra):
    """As close(), with infinities and what is no number in the same places."""
    got, want = got.double().cpu(), want.double()
    fine = want.isfinite()
    assert torch_equal(got.isnan(), want.isnan()) and torch_equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    close(got[fine], want[fine], size[fine], k, name, extra[fine])


def torch_equal(a, b):
    return a.shape == b.shape and bool((a == b).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,K,N,R", [(9, 64, 48, 8), (60, 136, 264, 16), (700, 192, 264, 64), (1500, 520, 1032, 24), (300, 71, 101, 7)])
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_infinities_of_adapters_stay_infinities(tf, torch, name, rows, K, N, R, how):
    # everything positive: an infinite factor gives that infinity in its column, whatever the middle's lower bits are
    rng = np.random.default_rng(rows)
    ids = rng.integers(-1, 3, rows)
    ids[:3] = [0, 1, 2]
    pos = lambda shape, scale=1.0: (tensor(torch, rng, shape, "float64").abs() * scale + 2.0 ** -6).to(getattr(torch, name))
    x, w, dy = pos((rows, K)), pos((K, N), K ** -0.5), pos((rows, N))
    a, b = pos((3, K, R), K ** -0.5), pos((3, R, N), R ** -0.5)
    inf = float("inf")
    bi = b.clone()
    bi[0, R - 1, 3], bi[1, 0, N - 2], bi[2, R // 2, 7] = inf, -inf, inf
    g = made(tf, torch, ids, 3)
    on = lambda *ts: [layout(torch, t, how) for t in ts]

    def plain(x, w, a, b):
        X, W, A, B = (t.double() for t in (x, w, a, b))
        y, size = X @ W, X @ W
        low = torch.zeros_like(y)
        for i in range(3):
            t = torch.from_numpy(np.nonzero(ids == i)[0])
            part = X[t] @ A[i] @ B[i]
            y[t] += part
            low[t] = part.abs()
        return y, size + low, low

    want, size, low = plain(x, w, a, bi)
    assert want.isinf().any() and not want.isnan().any()
    agree(tf.adapter_gemm(x.cuda(), *on(w, a, bi), g), want, size, K + R, name, MIDDLE[name] * low)
    # gradients: one infinite entry of x, one of dy, in rows of two groups
    xi, di = x.clone(), dy.clone()
    xi[0, 5], di[1, 6] = inf, inf
    dx, da, db = tf.adapter_gemm_backward(xi.cuda(), *on(w, a, b), di.cuda(), g)
    want, size, low = plain(di, w.t(), b.transpose(1, 2), a.transpose(1, 2))
    agree(dx, want, size, N + R, name, MIDDLE[name] * low)
    X, D, A, B = (t.double() for t in (xi, di, a, b))
    for i in range(3):
        t = torch.from_numpy(np.nonzero(ids == i)[0])
        want = X[t].t() @ (D[t] @ B[i].t())
        agree(da[i], want, want, len(t) + N, name, MIDDLE[name] * want)
        want = (X[t] @ A[i]).t() @ D[t]
        agree(db[i], want, want, len(t) + K, name, MIDDLE[name] * want)


# ------------------------------------------------------------------------------------------------------ what the sources have to keep to (no GPU)
def test_a_load_into_lds_writes_its_target_register_in_the_same_statement():
    # m0 says where the load goes: left to another statement, an instruction of the compiler's in between could change it
    import glob
    import re
    found = 0
    for path in glob.glob(os.path.join(ROOT, "tenferro-rs_amd", "csrc", "*.h*")):
        for text in re.findall(r"asm(?:\s+volatile)?\s*\((.*?)\);", open(path).read(), flags=re.S):
            code = " ".join(re.findall(r'"((?:[^"\\]|\\.)*)"', text.split("::")[0]))
            if re.search(r"buffer_load\w*.*\blds\b", code):
                found += 1
                assert re.search(r"\bm0\b.*buffer_load", code), (path, code)
            elif re.search(r"\bm0\b", code):
                raise AssertionError((path, code))
    assert found


# ------------------------------------------------------------------------------------------------------ calls that fail
@pytest.mark.gpu
def test_a_call_that_fails_on_another_stream_keeps_what_its_first_launch_uses(tf, torch, monkeypatch):
    x, up, down, ids, gates, dy = layer_inputs(torch, 3)
    groups = tf.RowGroups.from_ids(ids, up.shape[0])
    dc = torch.randn(groups.n_rows, up.shape[2], device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for call in ("tfh_ragged_gemm_grad", "tfh_adapter_gemm_grad"):
        before = len([e for e in tf._in_flight if not e[0].ready()])
        with monkeypatch.context() as m:
            m.setattr(tf.lib(), call, lambda *a: 2)
            with pytest.raises(tf.Error):
                if call == "tfh_ragged_gemm_grad":
                    tf.ragged_gemm_backward(x, up, dc, groups, gather=True, stream=side.cuda_stream)
                else:
                    flat = tf.RowGroups.from_ids(ids[:, 0], up.shape[0])
                    low_a, low_b = up[:, :, :8].contiguous(), up[:, :8, :].contiguous()
                    tf.adapter_gemm_backward(x, up[0].contiguous(), low_a, low_b, dc[:x.shape[0]].contiguous(), flat, stream=side.cuda_stream)
        held = tf._in_flight[-1][1]
        assert len(tf._in_flight) > before and any(t is x for t in held) and any(t is up for t in held) == (call == "tfh_ragged_gemm_grad")
        assert len([t for t in held if isinstance(t, torch.Tensor)]) >= 5      # operands, results and scratch
    side.synchronize()
    a = tf.ragged_gemm(x, up, groups, gather=True, stream=side.cuda_stream)     # and lets go of them
    torch.cuda.synchronize()
    assert len(tf._in_flight) <= 1 and torch.equal(a, tf.ragged_gemm(x, up, groups, gather=True))


@pytest.mark.gpu
def test_a_gradient_of_several_launches_looks_at_all_operands_first(tf, torch, monkeypatch):
    x, up, down, ids, gates, dy = layer_inputs(torch, 3)
    groups = tf.RowGroups.from_ids(ids, up.shape[0])
    dc = torch.zeros(groups.n_rows, up.shape[2], device="cuda")
    for name in ("tfh_ragged_gemm", "tfh_ragged_gemm_grad", "tfh_ragged_gemm_grad_a"):
        monkeypatch.setattr(tf.lib(), name, None)                               # nothing may be launched
    run = lambda a=x, b=up, d=dc, **k: tf.ragged_gemm_backward(a, b, d, groups, **dict(dict(gather=True), **k))
    for bad in (dict(a=x[1:]), dict(a=x[:, 1:]), dict(d=dc[1:]), dict(d=dc[:, 1:]), dict(b=up[1:]), dict(b=up[:, 1:]), dict(b=up[:, :, 1:]), dict(gather=False)):
        with pytest.raises(tf.ShapeMismatch):
            run(**bad)
    for bad in (dict(a=x[0]), dict(b=up[0]), dict(d=dc[0])):
        with pytest.raises(tf.RankMismatch):
            run(**bad)
    none = tf.RowGroups(groups.offsets, n_rows=groups.n_rows, fan=1)
    with pytest.raises(tf.InvalidArgument):
        tf.ragged_gemm_backward(torch.zeros(groups.n_rows, x.shape[1], device="cuda"), up, dc, none, gather=True)


@pytest.mark.gpu
def test_calls_on_a_side_stream_inside_a_capture_are_refused(tf, torch):
    # before anything is enqueued, so that the capture goes on; groups and Tensors from before it, with events, are taken
    x, up, down, ids, gates, dy = layer_inputs(torch, 12)
    want, groups, h = expert_layer(tf, x, up, down, ids, gates)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    st, T = side.cuda_stream, tf.Tensor.from_torch
    before = tf.RowGroups.from_ids(ids, up.shape[0], stream=st)
    held = T(x.clone())
    tf.ragged_gemm_into(T(x), T(up), before, 1.0, 0.0, T(torch.empty_like(h)), gather=True, stream=st)
    held.event = before.event
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: tf.RowGroups.from_ids(ids, up.shape[0], stream=st), lambda: tf.ragged_gemm(x, up, groups, gather=True, stream=st),
                     lambda: tf.combine_rows(h, groups, gates, stream=st)):
            with pytest.raises(tf.InvalidArgument):
                call()
        made_here = tf.RowGroups.from_ids(ids, up.shape[0], stream=torch.cuda.current_stream().cuda_stream)
        one = tf.ragged_gemm(x, up, before, gather=True)
        other = tf.ragged_gemm(held, T(up), made_here, gather=True)
        y = tf.combine_rows(tf.ragged_gemm(one, down, made_here), before, gates)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(one, h) and other.event is None
        assert np.array_equal(other.to_numpy(), h.cpu().numpy())
        z = tf.ragged_gemm(x, up, made_here, gather=True, stream=st)            # and outside, on the side stream
        torch.cuda.synchronize()
        assert torch.equal(z, h)


# ------------------------------------------------------------------------------------------------------ launches of many blocks
@pytest.mark.gpu
def test_joined_rows_of_more_tokens_than_one_grid_dimension_holds(tf, torch):
    # 2^26 tokens in blocks of four waves are 2^32 threads
    n, N = (1 << 26) + 5, 8
    x = torch.arange(n * N, dtype=torch.int32, device="cuda").remainder_(509).to(torch.bfloat16).view(n, N)      # exact, and others in every row
    positions = torch.arange(n, dtype=torch.int32, device="cuda")
    g = tf.RowGroups(torch.tensor([0, 7, n - 3], dtype=torch.int32, device="cuda"), positions, torch.where(positions < n - 3, positions, -1))
    y = tf.combine_rows(x, g)
    assert torch.equal(y[:n - 3], x[:n - 3]) and not y[n - 3:].any()
    weights = torch.full((n, 1), 2.0, device="cuda")
    dx, dw = tf.combine_rows_backward(x, weights, y, g)
    assert torch.equal(dx, y * 2) and bool((dw[n - 3:] == 0).all())
    some = torch.tensor([0, 1, 12345, (1 << 26) - 1, 1 << 26, n - 4], device="cuda")
    assert torch.equal(dw[some, 0].double(), (x[some].double() ** 2).sum(1))      # eight squares below 2^18: exact


@pytest.mark.gpu
def test_products_of_more_tiles_than_one_grid_dimension_holds(tf, torch):
    n = (1 << 30) + 333                                                           # 2^24 tiles of 64 rows, 256 threads each
    a = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(251).to(torch.bfloat16).view(n, 1)
    cut = 1000
    g = tf.RowGroups(torch.tensor([0, cut, n - 2], dtype=torch.int32, device="cuda"), n_rows=n)
    b = torch.tensor([2.0, -1.0], device="cuda").to(torch.bfloat16).view(2, 1, 1)
    c = tf.ragged_gemm(a, b, g)
    assert torch.equal(c[:cut], a[:cut] * 2) and torch.equal(c[cut:n - 2], -a[cut:n - 2]) and not c[n - 2:].any()
    del c
    groups = (1 << 24) + 77                                                       # and as many groups of a gradient
    x, d = a[:groups], a[100:100 + groups]
    g = tf.RowGroups(torch.arange(groups + 1, dtype=torch.int32, device="cuda"), n_rows=groups)
    out = torch.full((groups, 1, 1), float("nan"), dtype=torch.bfloat16, device="cuda")
    tf.ragged_gemm_grad_into(x, d, g, 1.0, 0.0, out)
    assert torch.equal(out.view(-1), (x.float() * d.float()).to(torch.bfloat16).view(-1))


def test_more_blocks_than_a_launch_has_are_refused(tf):
    L, V = tf.lib(), lambda *d: view(tf, d)
    for dt in (tf.BF16, tf.F64):
        refused(tf, L.tfh_ragged_gemm_grad(dt, row_groups(tf, n_rows=8, n_groups=1 << 30), 0, 1.0, V(8, 129), V(8, 129), 0.0, V(1 << 30, 129, 129), None), tf.InvalidArgument)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float32"])
@pytest.mark.parametrize("groups,each,K,N", [(2049, 3, 64, 72), (3000, 40, 35, 17), (5000, 0.01, 40, 24), (2500, 60, 72, 136), (100000, 2, 8, 8)])
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_products_of_many_groups(tf, torch, name, groups, each, K, N, how):
    # more groups than grouping by an index makes, some empty, with rows of none behind them; fewer rows than groups
    rng = np.random.default_rng(groups)
    counts = rng.integers(0, int(2 * each) + 1, groups) if each >= 1 else (rng.random(groups) < each).astype(int)
    counts[[0, -1]] = [0, 3]
    offsets = np.cumsum(np.concatenate([[0], counts]))
    n = int(offsets[-1]) + 5
    ids = torch.from_numpy(np.repeat(np.arange(groups), counts))
    g = tf.RowGroups(torch.from_numpy(offsets.astype(np.int32)).cuda(), n_rows=n)
    a, b, dc = tensor(torch, rng, (n, K), name), tensor(torch, rng, (groups, K, N), name, K ** -0.5), tensor(torch, rng, (n, N), name)
    A, B, D = (t.cuda().double() for t in (a, b, dc))
    on_b, p = layout(torch, b, how), slice(0, len(ids))
    chosen = ids.cuda()
    part = lambda x, m: torch.cat([torch.bmm(x[i:i + 4096, None], m[chosen[i:i + 4096]].contiguous())[:, 0] for i in range(0, len(ids), 4096)])
    got = tf.ragged_gemm(a.cuda(), on_b, g)
    close(got[p], part(A[p], B), part(A[p].abs(), B.abs()), K, name)
    assert not got[len(ids):].any()
    da, db = tf.ragged_gemm_backward(a.cuda(), on_b, dc.cuda(), g)
    Bt = B.transpose(1, 2).contiguous()
    close(da[p], part(D[p], Bt), part(D[p].abs(), Bt.abs()), N, name)
    assert not da[len(ids):].any()
    want, size = torch.zeros_like(B), torch.zeros_like(B)
    for i in range(0, len(ids), 4096):
        r = slice(i, min(i + 4096, len(ids)))
        outer = A[r, :, None] * D[r, None, :]
        want.index_add_(0, chosen[r], outer)
        size.index_add_(0, chosen[r], outer.abs())
    close(db, want, size, int(counts.max()), name)
    if groups < 10000:
        kept = torch.full((n, N), 7.0, dtype=a.dtype, device="cuda")                 # without zeros for the rows of none
        tf.ragged_gemm_into(a.cuda(), on_b, g, 1.0, 0.0, kept)
        assert torch.equal(kept[p], got[p]) and bool((kept[len(ids):] == 7).all())


@pytest.mark.gpu
def test_many_groups_that_do_not_ascend_stay_inside_the_views(tf, torch):
    # offsets of any order and size: results as they may be, accesses inside the rows
    rng = np.random.default_rng(5)
    for n in (40, 30000):
        offsets = rng.integers(-100, n + 100, 3001).astype(np.int32)
        g = tf.RowGroups(torch.from_numpy(offsets).cuda(), n_rows=n)
        a, b = torch.ones(n, 16, dtype=torch.bfloat16, device="cuda"), torch.ones(3000, 16, 8, dtype=torch.bfloat16, device="cuda")
        c = torch.zeros(n, 8, dtype=torch.bfloat16, device="cuda")
        tf.ragged_gemm_into(a, b, g, 1.0, 0.0, c)
        assert set(c.unique().tolist()) <= {0.0, 16.0}
        tf.ragged_gemm_backward(a, b, c, g)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------------ long sums of the 16-bit kernels
def device_products(torch, pairs):
    """[(x, y)] -> (sums, sums of absolute values) in 64 bits on the GPU."""
    return [(x @ y, x.abs() @ y.abs()) for x, y in ((x.cuda().double().contiguous(), y.cuda().double().contiguous()) for x, y in pairs)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16"])
@pytest.mark.parametrize("K,N", [(1032, 1544), (2568, 1288)])
@pytest.mark.parametrize("how", ["columns", "rows"])
@pytest.mark.parametrize("counts,tiles", [([6149], "256x256"), ([1100, 0, 700, 1], "256x128"), ([130, 190, 0, 61] * 5, "128x128"), ([40] * 40, "32x128")])
def test_long_sums_in_tiles_of_every_size(tf, torch, name, K, N, how, counts, tiles):
    # every slot of LDS is used many times over
    rng = np.random.default_rng(K + len(counts))
    offsets, rows = np.cumsum([0] + counts), sum(counts)
    a, b = tensor(torch, rng, (rows, K), name), tensor(torch, rng, (len(counts), K, N), name, K ** -0.5)
    g = tf.RowGroups(torch.tensor(offsets, dtype=torch.int32, device="cuda"), n_rows=rows)
    got = tf.ragged_gemm(a.cuda(), layout(torch, b, how), g)
    assert tiles in tf.last_kernel() and "fast" in tf.last_kernel(), tf.last_kernel()
    cut = [slice(offsets[i], offsets[i + 1]) for i in range(len(counts))]
    for s, (want, size) in zip(cut, device_products(torch, [(a[s], b[i]) for i, s in enumerate(cut)])):
        close(got[s], want, size, K, name)
    if len(counts) < 40:
        dc = tensor(torch, rng, (rows, N), name)
        da, db = tf.ragged_gemm_backward(a.cuda(), layout(torch, b, how), dc.cuda(), g)
        for s, (want, size) in zip(cut, device_products(torch, [(dc[s], b[i].t()) for i, s in enumerate(cut)])):
            close(da[s], want, size, N, name)
        for i, (want, size) in enumerate(device_products(torch, [(a[s].t(), dc[s]) for s in cut])):
            close(db[i], want, size, max(counts), name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16"])
@pytest.mark.parametrize("K", [2056, 4104])
@pytest.mark.parametrize("counts", [[4, 0, 3, 1], [20, 17], [50, 49, 0], [1]], ids=str)
def test_long_sums_of_few_rows(tf, torch, name, K, counts):
    rng = np.random.default_rng(K + sum(counts))
    N, offsets, rows = 264, np.cumsum([0] + counts), sum(counts)
    a, b = tensor(torch, rng, (rows, K), name), tensor(torch, rng, (len(counts), K, N), name, K ** -0.5)
    g = tf.RowGroups(torch.tensor(offsets, dtype=torch.int32, device="cuda"), n_rows=rows)
    got = tf.ragged_gemm(a.cuda(), layout(torch, b, "rows"), g)
    assert "few" in tf.last_kernel(), tf.last_kernel()
    cut = [slice(offsets[i], offsets[i + 1]) for i in range(len(counts))]
    for s, (want, size) in zip(cut, device_products(torch, [(a[s], b[i]) for i, s in enumerate(cut)])):
        close(got[s], want, size, K, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,groups,K,N,R", [(8, 2, 4104, 520, 16), (20, 3, 4104, 1032, 64), (64, 5, 4104, 4104, 128), (500, 3, 4104, 1032, 16), (500, 3, 1032, 4104, 64), (500, 2, 4104, 1032, 128), (4480, 64, 1032, 1032, 32), (9000, 16, 1096, 520, 24)])
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_long_sums_of_adapters(tf, torch, name, tokens, groups, K, N, R, how):
    rng = np.random.default_rng(tokens + K + R)
    ids = rng.integers(-1, groups, tokens)
    x, dy, w = tensor(torch, rng, (tokens, K), name), tensor(torch, rng, (tokens, N), name), tensor(torch, rng, (K, N), name, K ** -0.5)
    a, b = tensor(torch, rng, (groups, K, R), name, K ** -0.5), tensor(torch, rng, (groups, R, N), name, R ** -0.5)
    scales = torch.from_numpy(0.2 + rng.random(groups)).float()
    g = made(tf, torch, ids, groups)
    on = [layout(torch, t, how) for t in (w, a, b)]
    y = tf.adapter_gemm(x.cuda(), *on, g, scales.cuda())
    dx, da, db = tf.adapter_gemm_backward(x.cuda(), *on, dy.cuda(), g, scales.cuda())
    X, D, W, A, B, S = (t.cuda().double() for t in (x, dy, w, a, b, scales))
    wt = W.t().contiguous()
    want_y, size_y, want_x, size_x = X @ W, X.abs() @ W.abs(), D @ wt, D.abs() @ wt.abs()
    low_y, low_x = torch.zeros_like(want_y), torch.zeros_like(want_x)
    for i in range(groups):
        t = torch.from_numpy(np.nonzero(ids == i)[0]).cuda()
        x_, d_, at, bt = X[t], D[t], A[i].t().contiguous(), B[i].t().contiguous()
        v, u, va, ua = x_ @ A[i], d_ @ bt, x_.abs() @ A[i].abs(), d_.abs() @ bt.abs()
        want_y[t] += S[i] * (v @ B[i])
        low_y[t] = S[i] * (va @ B[i].abs())
        want_x[t] += S[i] * (u @ at)
        low_x[t] = S[i] * (ua @ at.abs())
        xt, vt = x_.t().contiguous(), v.t().contiguous()
        size = S[i] * (xt.abs() @ ua)
        close(da[i], S[i] * (xt @ u), size, len(t) + N, name, MIDDLE[name] * size.cpu())
        size = S[i] * (va.t().contiguous() @ d_.abs())
        close(db[i], S[i] * (vt @ d_), size, len(t) + K, name, MIDDLE[name] * size.cpu())
    close(y, want_y, size_y + low_y, K + R, name, MIDDLE[name] * low_y.cpu())
    close(dx, want_x, size_x + low_x, N + R, name, MIDDLE[name] * low_x.cpu())


# ------------------------------------------------------------------------------------------------------ the middle product of f16 adapters
@pytest.mark.gpu
@pytest.mark.parametrize("rows,K,N,R", [(30, 64, 48, 8), (60, 520, 264, 16), (700, 192, 264, 64), (300, 1032, 520, 128)])
@pytest.mark.parametrize("apart", [0, 12, 24])
@pytest.mark.parametrize("how", ["columns", "rows"])
def test_the_middle_of_f16_adapters_keeps_22_bits(tf, torch, rows, K, N, R, apart, how):
    # Its elements are kept to half of 2^-21 of their own size, and to half of f16's smallest step, 2^-24, where the row's largest is at
    # least 2^14 of these: 2^-39 of it.  Every second column of a is 2^-apart as large as the others, whose rows of b do the same: each
    # contributes as much.  With w = 0 nothing covers for it.
    rng = np.random.default_rng(rows + apart)
    ids = rng.integers(-1, 3, rows)
    x, w = tensor(torch, rng, (rows, K), "float16"), torch.zeros(K, N, dtype=torch.float16)
    up, down = 2.0 ** min(apart, 10), 2.0 ** -max(0, apart - 10)
    big = torch.where(torch.arange(R) % 2 == 0, up, down)
    a = (torch.from_numpy(rng.standard_normal((3, K, R))) * K ** -0.5 * big).to(torch.float16)
    b = (torch.from_numpy(rng.standard_normal((3, R, N))) / big[:, None] * up * 2.0 ** -min(apart, 10)).clamp(-6e4, 6e4).to(torch.float16)      # in range
    if apart == 24:
        b[:, ::2] = 0                                        # the small ones alone
    on = [layout(torch, t, how) for t in (w, a, b)]
    got = tf.adapter_gemm(x.cuda(), *on, made(tf, torch, ids, 3))
    want, size, low = adapter_reference(torch, x, w, a, b, None, ids)
    extra = 2.0 ** -22 * low
    for i in range(3):
        t = torch.from_numpy(np.nonzero(ids == i)[0])
        v = x[t].double() @ a[i].double()
        extra[t] += 2.0 ** -39 * v.abs().max(1, keepdim=True).values * b[i].double().abs().sum(0)
    close(got, want, size, K + R, "float16", extra)


# ------------------------------------------------------------------------------------------------------ what a torch tensor may carry beside its values
@pytest.mark.gpu
def test_tensors_with_the_negative_bit_are_refused(tf, torch):
    # .conj().imag is a real tensor whose memory holds the values with the other sign
    z = torch.randn(8, 16, dtype=torch.complex64, device="cuda")
    neg = z.conj().imag
    assert neg.is_neg()
    x, w = torch.randn(8, 16, device="cuda"), torch.randn(2, 16, 4, device="cuda")
    g = tf.RowGroups(torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda"), n_rows=8)
    placed = tf.RowGroups.from_ids(torch.zeros(8, dtype=torch.int64, device="cuda"), 2)
    for call in (lambda: tf.ragged_gemm(neg, w, g), lambda: tf.ragged_gemm(x, neg.unflatten(1, (4, 4)).permute(1, 0, 2)[:2], g), lambda: tf.combine_rows(neg, placed),
                 lambda: tf.combine_rows(x, placed, neg[:, :1]), lambda: tf.adapter_gemm(neg, w[0], w[:, :, :2], w[:, :2], placed),
                 lambda: tf.ragged_gemm_into(x, w, g, 1.0, 0.0, neg[:, :4]), lambda: tf.Tensor.from_torch(neg)):
        with pytest.raises(tf.InvalidArgument, match="negative bit"):
            call()
    same = tf.ragged_gemm(neg.resolve_neg(), w, g)
    assert torch.equal(same, tf.ragged_gemm((-z.imag).contiguous(), w, g))


@pytest.mark.gpu
def test_operands_of_autograd_are_refused_where_a_gradient_would_go_missing(tf, torch):
    x, w = torch.randn(8, 16, device="cuda"), torch.randn(2, 16, 4, device="cuda")
    g = tf.RowGroups(torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda"), n_rows=8)
    placed = tf.RowGroups.from_ids(torch.zeros(8, 1, dtype=torch.int64, device="cuda"), 2)
    gates = torch.ones(8, 1, device="cuda")
    want = tf.ragged_gemm(x, w, g)
    leaf = torch.nn.Parameter(w.clone())
    for call in (lambda: tf.ragged_gemm(x, leaf, g), lambda: tf.ragged_gemm(x.clone().requires_grad_(), w, g), lambda: tf.combine_rows(x, placed, gates.clone().requires_grad_()),
                 lambda: tf.adapter_gemm(x, leaf[0], w[:, :, :2], w[:, :2], placed)):
        with pytest.raises(tf.InvalidArgument, match="requires grad"):
            call()
        with torch.no_grad():
            call()
    with torch.inference_mode():
        assert torch.equal(tf.ragged_gemm(x, leaf, g), want)

    class Ragged(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a, b):
            ctx.save_for_backward(a, b)
            return tf.ragged_gemm(a, b, g)

        @staticmethod
        def backward(ctx, dc):
            return tf.ragged_gemm_backward(*ctx.saved_tensors, dc, g)

    a = x.clone().requires_grad_()
    y = Ragged.apply(a, leaf)
    dy = torch.randn_like(y)
    da, db = torch.autograd.grad(y, (a, leaf), dy)
    wa, wb = tf.ragged_gemm_backward(x, w, dy, g)
    assert torch.equal(y.detach(), want) and torch.equal(da, wa) and torch.equal(db, wb)
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        assert torch.equal(tf.ragged_gemm(x, w, g), want)
        with pytest.raises(tf.InvalidArgument, match="dual"):
            tf.ragged_gemm(fw.make_dual(x, torch.ones_like(x)), w, g)


# ------------------------------------------------------------------------------------------------------ choices taken out after grouping
@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bfloat16", "float32"])
@pytest.mark.parametrize("tokens,fan,groups,N", [(1, 1, 1, 3), (40, 2, 5, 64), (700, 4, 8, 24), (9000, 2, 6, 40)])
@pytest.mark.parametrize("listed", [True, False])
def test_choices_whose_position_was_taken_out_get_no_gradient(tf, torch, name, tokens, fan, groups, N, listed):
    # a capacity limit applied to the positions: the rows still stand in their groups, and no token reads them
    rng = np.random.default_rng(tokens)
    ids = choices(rng, tokens, fan, groups)
    if not listed:
        ids = np.where((ids < 0) | (ids >= groups), groups, ids)
        ids = np.sort(ids.reshape(-1)).reshape(tokens, fan)          # rows that lie in order: no order is given
    offsets, order, positions = grouping(ids.reshape(-1), groups)
    assert listed or order == list(range(tokens * fan))
    positions, n = np.asarray(positions), tokens * fan
    positions[rng.random(n) < 0.4] = -1
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")
    g = tf.RowGroups(i32(offsets), i32(order) if listed else None, i32(positions), n_rows=n, fan=fan)
    x, dy = tensor(torch, rng, (n, N), name), tensor(torch, rng, (tokens, N), name)
    w = torch.from_numpy(rng.standard_normal((tokens, fan))).float()
    junk = torch.full((n, N), float("nan"), dtype=x.dtype, device="cuda")
    del junk                                                         # what the next buffer of that size finds there
    dx, dw = tf.combine_rows_backward(x.cuda(), w.cuda(), dy.cuda(), g)
    want, size = torch.zeros(n, N, dtype=torch.float64), torch.zeros(tokens * fan, dtype=torch.float64)
    want_w = torch.zeros(tokens * fan, dtype=torch.float64)
    kept = torch.from_numpy(np.nonzero(positions >= 0)[0])
    p = torch.from_numpy(positions[positions >= 0])
    want[p] = w.reshape(-1)[kept, None].double() * dy[kept // fan].double()
    want_w[kept] = (x[p].double() * dy[kept // fan].double()).sum(1)
    size[kept] = (x[p].double() * dy[kept // fan].double()).abs().sum(1)
    close(dx, want, want.abs(), 1, name)
    close(dw.reshape(-1), want_w, size, N, "float32")


@pytest.mark.gpu
@pytest.mark.parametrize("name,K,N,rows", [("bfloat16", 64, 64, 900), ("float16", 256, 520, 9000), ("bfloat16", 4104, 264, 30), ("float32", 33, 5, 40), ("bfloat16", 35, 17, 300)])
def test_rows_of_no_group_are_zeros_whatever_the_factor(tf, torch, name, K, N, rows):
    code = {"bfloat16": tf.BF16, "float16": tf.F16, "float32": tf.F32}[name]
    dtype = getattr(torch, name)
    a, b, c = torch.ones(rows, K, dtype=dtype, device="cuda"), torch.ones(2, N, K, dtype=dtype, device="cuda").transpose(1, 2), torch.ones(rows, N, dtype=dtype, device="cuda")
    g = tf.RowGroups(torch.tensor([0, 3, rows // 2], dtype=torch.int32, device="cuda"), n_rows=rows)
    at = lambda t: view(tf, list(t.shape), list(t.stride()), t.data_ptr())
    for alpha in (float("inf"), float("nan")):
        tf._check(tf.lib().tfh_ragged_gemm(code, C.byref(g._c), 4, alpha, at(a), at(b), 0.0, at(c), torch.cuda.current_stream().cuda_stream))
        assert not c[rows // 2:].any() and not c[:rows // 2].isfinite().any()


@pytest.mark.parametrize("make", ["zeros", "ones", "empty"])
def test_main_memory_refuses_bf16_by_name(tf, make):
    with pytest.raises(tf.InvalidArgument, match="bf16"):
        getattr(tf.Tensor, make)([2, 3], tf.MainMemory, tf.MemoryOrder.RowMajor, tf.BF16)
    assert getattr(tf.Tensor, make)([2, 3], tf.MainMemory, tf.MemoryOrder.RowMajor, tf.F16).to_numpy().dtype == np.float16


@pytest.mark.gpu
def test_bf16_does_not_move_to_main_memory(tf, torch):
    t = tf.Tensor.from_torch(torch.ones(2, 3, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(tf.InvalidArgument, match="bf16"):
        t.to_memory_space_async(tf.MainMemory)
    assert t.to_numpy().tolist() == [[1.0] * 3] * 2


@pytest.mark.gpu
def test_numbers_that_32_bit_fields_do_not_hold_are_refused(tf, torch):
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    for n in (0, -1, 2049, 1 << 31, (1 << 32) + 4):
        with pytest.raises(tf.InvalidArgument):
            tf.RowGroups.from_ids(ids, n)
    offsets = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    for k in (dict(n_rows=0, fan=(1 << 32) + 1), dict(n_rows=1 << 40), dict(n_rows=(1 << 32), fan=1 << 32), dict(n_rows=-1), dict(n_rows=0, fan=0)):
        with pytest.raises(tf.InvalidArgument):
            tf.RowGroups(offsets, **k)


@pytest.mark.gpu
def test_gradients_of_tensors_are_laid_out_like_them(tf, torch):
    x, up, down, ids, gates, dy = layer_inputs(torch, 15)
    T, flat = tf.Tensor.from_torch, tf.RowGroups.from_ids(ids[:, 0], up.shape[0])
    dc = torch.randn(x.shape[0], up.shape[2], device="cuda")
    want = tf.ragged_gemm_backward(x, up, dc, flat, gather=True)
    columns = up.transpose(1, 2).contiguous().transpose(1, 2)
    order = tf.Tensor(up.permute(2, 1, 0).contiguous().view(-1), list(up.shape), [1, up.shape[0], up.shape[0] * up.shape[1]], 0, tf.GpuMemory(0), tf.F32)   # column-major
    big = torch.zeros(up.numel() + 7, device="cuda")
    big[5:5 + up.numel()].copy_(up.reshape(-1))
    shifted = tf.Tensor(big, list(up.shape), list(up.stride()), 5, tf.GpuMemory(0), tf.F32)
    for b in (T(up), T(columns), order, shifted, T(up).permute([0, 2, 1]).permute([0, 2, 1])):
        da, db = tf.ragged_gemm_backward(T(x), b, T(dc), flat, gather=True)
        assert db.strides() == b.strides()
        close(torch.from_numpy(db.to_numpy()), want[1], want[1].abs() + 10, 48, "float32")
        assert np.abs(da.to_numpy() - want[0].cpu().numpy()).max() < 1e-4
    wide = T(up[:1].expand(up.shape[0], -1, -1))                          # one matrix for all groups: nothing to be laid out like
    _, db = tf.ragged_gemm_backward(T(x), wide, T(dc), flat, gather=True)
    assert db.dims() == list(up.shape) and 0 not in db.strides()


def test_buffers_held_by_another_thread_meanwhile_stay_held(tf, monkeypatch):
    # asking an event lets other threads run: what they add to the list of buffers in use stays in it
    class Event:
        def __init__(self, done, then=None):
            self.done, self.then = done, then

        def ready(self):
            if self.then:
                self.then()
            return self.done

    kept = []
    monkeypatch.setattr(tf, "_in_flight", kept)
    meanwhile = lambda: kept.append((Event(False), ["theirs"])) if not any(e[1] == ["theirs"] for e in kept) else None
    gone = (Event(True), ["taken out by the other"])
    kept += [(Event(True, meanwhile), ["done"]), (Event(False, lambda: kept.remove(gone) if gone in kept else None), ["running"]), gone]
    tf._hold(Event(False), ["ours"])
    assert [e[1] for e in kept] == [["running"], ["theirs"], ["ours"]]
