"""Text-model operators (ops.embedding_sorted, ops.linear_cross_entropy, optim.clip_grads) against their definitions in 64 bits.

Tolerances are bounds, element by element, from the roundings that the kernels make: u = 2^-24 for each fp32 operation, half an
epsilon of the output's type (bf16 2^-8, fp32 2^-24) for each rounding to it."""
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(__file__), 'golden'))

EMU = os.environ.get('S2AG_EMU', '0') == '1'
U = 2.0 ** -24
DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}


@pytest.fixture(scope='module')
def S():
    from speech2affective_gestures_amd import _lib, ops, optim
    return dict(ops=ops, optim=optim, lib=_lib)


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, ref, bound):
    got, ref, bound = got.detach().cpu().double(), ref.double(), bound.double()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all()
    over = (got - ref).abs() - bound
    worst = int(over.argmax()) if over.numel() else 0
    assert over.numel() == 0 or float(over.max()) <= 0, (worst, got.reshape(-1)[worst], ref.reshape(-1)[worst], bound.reshape(-1)[worst])


# ---- embedding --------------------------------------------------------------------------------------------------------------
def embedding_reference(ids, table, dy, scale, padding_idx, dtype):
    """(y, bound), (dtable, bound) on the CPU in 64 bits."""
    n_entries, dim = table.shape
    flat = ids.reshape(-1)
    ok = (flat >= 0) & (flat < n_entries)
    at = torch.where(ok, flat, torch.zeros_like(flat))
    y = table.double()[at] * scale * ok[:, None]
    h = half_eps(dtype)
    y_bound = y.abs() * (U + h * (1 + U))                                   # one product, one rounding
    if padding_idx is not None:
        ok = ok & (flat != padding_idx)
    g = dy.double().reshape(-1, dim) * ok[:, None]
    dt = torch.zeros(n_entries, dim, dtype=torch.float64).index_add_(0, at, g)
    s = torch.zeros(n_entries, dim, dtype=torch.float64).index_add_(0, at, g.abs()) * abs(scale)
    m = torch.zeros(n_entries, dtype=torch.float64).index_add_(0, at, ok.double())[:, None]
    dt *= scale
    err = s * (m + 2) * U * 1.01                                            # m - 1 sums and a product, in any order
    return (y.reshape(*ids.shape, dim), y_bound.reshape(*ids.shape, dim)), (dt, err + h * (dt.abs() + err))


def ids_of(kind, n, entries, g):
    ids = torch.randint(0, entries, (n,), generator=g)
    if kind == 'padded':                       # transcripts: most positions hold one id
        ids[torch.rand(n, generator=g) < 0.85] = 0
    elif kind == 'one':
        ids[:] = entries - 1
    elif kind == 'runs':
        ids = ids.sort().values
    elif kind == 'outside':
        ids[::3] = -1
        ids[1::5] = entries
    return ids


# (positions, dim, rows of the table): around the lengths of a tile (16, 64), of the two sorts (8192; 4096), of a vector and a chunk of columns
EMB_CASES = [(1, 1, 1), (1, 8, 3), (2, 300, 2), (15, 7, 40), (16, 64, 16), (17, 64, 16), (33, 257, 5), (64, 512, 700), (136, 300, 2000),
             (1000, 36, 255), (1023, 5, 256), (1025, 5, 257), (4097, 12, 65537), (8192, 4, 90), (8193, 4, 511), (8193, 9, 140000), (12289, 16, 513)]


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('kind', ['even', 'padded', 'one', 'outside'])
@pytest.mark.parametrize('case', EMB_CASES)
def test_embedding_sorted(S, case, kind, dtype):
    n, dim, entries = case
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(n * 7 + dim + entries)
    ids = ids_of(kind, n, entries, g)
    table, dy = torch.randn(entries, dim, generator=g).to(dt), torch.randn(n, dim, generator=g).to(dt)
    scale = math.sqrt(dim)
    (y, yb), (gr, gb) = embedding_reference(ids, table, dy, scale, None, dt)
    t = table.cuda().requires_grad_(True)
    out = S['ops'].embedding_sorted(ids.cuda(), t, scale=scale)
    assert out.dtype == dt
    within(out, y, yb)
    out.backward(dy.cuda())
    assert t.grad.dtype == dt
    within(t.grad, gr, gb)
    first = t.grad.clone()                      # the same bits again
    t.grad = None
    S['ops'].embedding_sorted(ids.cuda(), t, scale=scale).backward(dy.cuda())
    assert torch.equal(first, t.grad)


@pytest.mark.parametrize('tile,dim,dtype', [(16, 20, 'fp32'), (16, 600, 'bf16'),
                                            pytest.param(64, 4100, 'fp32', marks=pytest.mark.skipif(EMU, reason='a hundred million values'))])
def test_embedding_sorted_runs_that_end_with_a_tile(S, tile, dim, dtype):
    """Runs of equal ids that begin and end at borders of the tiles the sums go by, one short of them and one behind, across one tile
    to more than 64 of them."""
    tiles = [1, 1, 2, 3, 15, 16, 17, 63, 64, 65, 66, 130]
    lengths = [tile * k for k in tiles] + [5] + [tile * k - 1 for k in tiles] + [tile * k + 1 for k in tiles] + [tile * k for k in tiles]
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(tile + dim)
    ids = torch.arange(len(lengths)).repeat_interleave(torch.tensor(lengths))
    ids = ids[torch.randperm(ids.numel(), generator=g)]
    table, dy = torch.randn(len(lengths), dim, generator=g).to(dt), torch.randn(ids.numel(), dim, generator=g).to(dt)
    _, (gr, gb) = embedding_reference(ids, table, dy, 1.0, None, dt)
    t = table.cuda().requires_grad_(True)
    S['ops'].embedding_sorted(ids.cuda(), t).backward(dy.cuda())
    within(t.grad, gr, gb)


def test_embedding_sorted_padding_row_shapes_and_small_ids(S):
    g = torch.Generator().manual_seed(3)
    ids = ids_of('padded', 6 * 35, 50, g).view(6, 35)
    table, dy = torch.randn(50, 24, generator=g), torch.randn(6, 35, 24, generator=g)
    for pad in (0, -50, 7):
        (y, yb), (gr, gb) = embedding_reference(ids, table, dy, 1.0, pad % 50, torch.float32)
        t = table.cuda().requires_grad_(True)
        out = S['ops'].embedding_sorted(ids.to(torch.int32).cuda(), t, padding_idx=pad)
        within(out, y, yb)
        out.backward(dy.cuda())
        within(t.grad, gr, gb)
        assert float(t.grad[pad % 50].abs().max()) == 0.0


@pytest.mark.parametrize('dtype', list(DTYPES))
def test_embedding_sorted_strides_and_offsets(S, dtype):
    """ids and dy that are slices, transposed or broadcast; a table that does not begin at a multiple of 16 bytes."""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(5)
    wide = torch.randint(0, 30, (9, 40), generator=g)
    ids = wide[:, 3:37].t()
    flat = torch.randn(30 * 16 + 1, generator=g).to(dt)
    table = flat[1:].view(30, 16)
    dy_wide = torch.randn(34, 9, 20, generator=g).to(dt)
    for dy in (dy_wide[:, :, 2:18], dy_wide[:, :, 4:20], dy_wide[:, :1, :16].expand(34, 9, 16), dy_wide[:, :, :1].expand(34, 9, 16)):
        (y, yb), (gr, gb) = embedding_reference(ids, table, dy, 2.0, None, dt)
        t = flat.cuda()[1:].view(30, 16).requires_grad_(True)
        base = dy_wide.cuda()
        dyc = torch.as_strided(base, dy.shape, dy.stride(), dy.storage_offset())
        out = S['ops'].embedding_sorted(wide.cuda()[:, 3:37].t(), t, scale=2.0)
        within(out, y, yb)
        (grad,) = torch.autograd.grad(out, t, dyc)
        within(grad, gr, gb)


def test_embedding_sorted_no_ids_and_rows_without_an_id(S):
    t = torch.randn(40, 12, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    out = S['ops'].embedding_sorted(torch.zeros(3, 0, dtype=torch.int64).cuda(), t)
    assert out.shape == (3, 0, 12)
    out.sum().backward()
    assert float(t.grad.abs().max()) == 0.0
    t.grad = None
    out = S['ops'].embedding_sorted(torch.full((70,), -5).cuda(), t)
    assert float(out.abs().max()) == 0.0
    out.sum().backward()
    assert float(t.grad.abs().max()) == 0.0


def test_embedding_sorted_adds_to_the_arena(S):
    """A table of a ParamArena: the backward pass adds to its gradient there; other rows and other parameters stay as they are."""
    g = torch.Generator().manual_seed(9)
    table, other = torch.randn(60, 20, generator=g), torch.randn(7, generator=g)
    ids, dy = ids_of('padded', 90, 50, g), torch.randn(90, 20, generator=g)
    a, b = torch.nn.Parameter(table.cuda()), torch.nn.Parameter(other.cuda())
    arena = S['optim'].ParamArena([a, b])
    start = torch.randn(arena.numel, generator=g)
    arena.grad.copy_(start.cuda())
    _, (gr, gb) = embedding_reference(ids, table, dy, 0.5, None, torch.float32)
    S['ops'].embedding_sorted(ids.cuda(), a, scale=0.5).backward(dy.cuda())
    before = start[:1200].view(60, 20).double()
    within(a.grad, before + gr, gb + U * (before.abs() + gr.abs() + gb) * 1.01)
    assert torch.equal(a.grad.cpu()[50:], start[:1200].view(60, 20)[50:])
    assert torch.equal(arena.grad.cpu()[1200:], start[1200:])


def test_embedding_sorted_refusals(S):
    f = S['ops'].embedding_sorted
    ids, table = torch.zeros(4, dtype=torch.int64).cuda(), torch.zeros(5, 6).cuda()
    for a, kw, err in [((ids.float(), table), {}, TypeError), ((ids, table.double()), {}, TypeError), ((ids, table.half()), {}, TypeError),
                       ((ids, table[0]), {}, ValueError), ((ids, table[:0]), {}, ValueError), ((ids, table[:, :0]), {}, ValueError),
                       ((ids, table), dict(padding_idx=5), ValueError), ((ids, table), dict(padding_idx=-6), ValueError), ((None, table), {}, TypeError)]:
        with pytest.raises(err):
            f(*a, **kw)


# ---- linear cross entropy ----------------------------------------------------------------------------------------------------
IGNORE = -100


def lce_reference(x, w, target, gout, reduction, ignore=IGNORE):
    """(loss, bound), (dx, bound), (dw, bound) in 64 bits.  The bounds follow the kernels: a logit is a sum of `terms` fp32 terms;
    an exponential of an argument of size s is off by s u + 4 u of itself (its argument's product with log2 e, its own rounding);
    G is rounded to bf16 for bf16 operands, its and the other operand's pieces carry 2^-23 for fp32.  fp32 logits are three products of
    two halves each: a value's second half leaves 2^-11 of the 2^-11 that the first left, 2^-22 = 4 u of it, and the product of the
    second halves, another 2^-22, is left out: 12 u of |x| |w| in all.  A value below 2^-17 of its row's
    largest keeps less, 2^-39 of that largest one: no test has such columns together with words that make them count."""
    dt = x.dtype
    pieces = 6 if dt == torch.float32 else 1
    x64, w64 = x.double(), w.double()
    n, d = x.shape
    z = x64 @ w64.t()
    za = (x64.abs() @ w64.abs().t()).max() if n else torch.tensor(0.0)
    dz = float(za) * ((d * min(pieces, 3) + 4) * U + (12 * U if pieces > 1 else 0))  # sums; what the halves leave
    keep = target != ignore
    at = torch.where(keep, target, torch.zeros_like(target)).long()
    lse = torch.logsumexp(z, 1)
    spread = float(z.max() - z.min()) + dz if n else 0.0
    de = (2 * spread + 16 + w.shape[0] ** 0.5) * U                                  # exponentials, their sum in steps, the joins
    dl = 2 * dz + de + 4 * U * (float(lse.abs().max()) if n else 0.0)
    loss = (lse - z[torch.arange(n), at]) * keep
    loss_bound = (dl + 2 * U * (lse.abs() + loss.abs())) * keep
    m = int(keep.sum())
    f = {'mean': gout / max(m, 1), 'sum': gout, 'none': gout}[reduction]
    f = f.double() * keep                                                            # (rows,)
    p = torch.softmax(z, 1)
    one = torch.zeros_like(p)
    one[torch.arange(n), at] = 1.0
    g = (p - one) * f[:, None]
    ga = p * f.abs()[:, None] * (dl + de + dz) * 1.1 + g.abs() * 4 * U               # G in fp32
    ga = ga + (g.abs() + ga) * (half_eps(torch.bfloat16) if pieces == 1 else 4 * U)  # as the products read it
    h = half_eps(dt)

    def product(a, da, b, terms):
        r = a @ b
        e = da @ b.abs() + (a.abs() + da) @ b.abs() * ((terms * pieces + 8) * U)
        return r, e + h * (r.abs() + e)
    dx, dxb = product(g, ga, w64, w.shape[0])
    dw, dwb = product(g.t(), ga.t(), x64, n)
    if reduction == 'none':
        return (loss, loss_bound), (dx, dxb), (dw, dwb)
    s, sb = loss.sum(), loss_bound.sum()
    if reduction == 'mean':
        s, sb = s / max(m, 1), sb / max(m, 1)
    return (s, sb + 2 * U * s.abs()), (dx, dxb), (dw, dwb)


def lce_case(n, d, v, dtype, ignored, seed=0):
    g = torch.Generator().manual_seed(n * 31 + d * 7 + v + seed)
    x, w = torch.randn(n, d, generator=g).to(DTYPES[dtype]), (torch.randn(v, d, generator=g) * 2 / math.sqrt(d)).to(DTYPES[dtype])
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.rand(n, generator=g) < ignored] = IGNORE
    return x, w, t, g


def lce_check(S, x, w, t, g, reduction):
    gout = torch.randn(t.shape if reduction == 'none' else (), generator=g)
    (l, lb), (dx, dxb), (dw, dwb) = lce_reference(x, w, t, gout, reduction)
    xg, wg, tg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True), t.cuda()
    loss = S['ops'].linear_cross_entropy(xg, wg, tg, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == l.shape
    within(loss, l, lb)
    loss.backward(gout.cuda())
    within(xg.grad, dx, dxb)
    within(wg.grad, dw, dwb)
    again = torch.autograd.grad(S['ops'].linear_cross_entropy(xg, wg, tg, reduction=reduction), (xg, wg), gout.cuda())
    assert torch.equal(again[0], xg.grad) and torch.equal(again[1], wg.grad)


# (rows, dim, words): one of each, around a stage of k (64), the tiles (128, 256), a transposed block, an odd pitch
LCE_CASES = [(1, 1, 1), (1, 64, 2), (2, 8, 300), (3, 300, 129), (17, 65, 257), (64, 63, 1000), (127, 128, 128), (129, 130, 511), (257, 64, 513),
             (300, 36, 2049), (136, 300, 1000)]


@pytest.mark.parametrize('ignored', [0.0, 0.6])
@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('case', LCE_CASES)
def test_linear_cross_entropy(S, case, dtype, ignored):
    x, w, t, g = lce_case(*case, dtype, ignored)
    lce_check(S, x, w, t, g, 'mean')


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('reduction', ['sum', 'none'])
def test_linear_cross_entropy_reductions(S, reduction, dtype):
    x, w, t, g = lce_case(70, 96, 333, dtype, 0.3)
    lce_check(S, x, w, t, g, reduction)


@pytest.mark.skipif(EMU, reason='hundreds of large tiles: minutes on the device model')
@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('case', [(250, 64, 65536), (65530, 40, 300), (1100, 520, 50021), (1000, 520, 65536), (4100, 800, 700),
                                  (40, 800, 30000)])
def test_linear_cross_entropy_large_tiles(S, case, dtype):
    x, w, t, g = lce_case(*case, dtype, 0.2)
    lce_check(S, x, w, t, g, 'mean')


@pytest.mark.skipif(EMU, reason='hundreds of large tiles: minutes on the device model')
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_linear_cross_entropy_in_pieces_of_the_vocabulary(S, dtype):
    """More rows times words than one piece holds."""
    n, d, v = 20000, 8, 13501
    x, w, t, g = lce_case(n, d, v, dtype, 0.1)
    lce_check(S, x, w, t, g, 'mean')


@pytest.mark.parametrize('dtype', list(DTYPES))
def test_linear_cross_entropy_all_rows_ignored(S, dtype):
    x, w, t, g = lce_case(40, 24, 77, dtype, 0.0)
    t[:] = IGNORE
    for reduction in ('mean', 'sum', 'none'):
        xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        loss = S['ops'].linear_cross_entropy(xg, wg, t.cuda(), reduction=reduction)
        assert float(loss.abs().max()) == 0.0
        loss.sum().backward()
        assert float(xg.grad.abs().max()) == 0.0 and float(wg.grad.abs().max()) == 0.0


def test_linear_cross_entropy_no_rows(S):
    x, w = torch.zeros(0, 24).cuda().requires_grad_(True), torch.randn(77, 24).cuda().requires_grad_(True)
    for reduction in ('mean', 'sum', 'none'):
        loss = S['ops'].linear_cross_entropy(x, w, torch.zeros(0, dtype=torch.int64).cuda(), reduction=reduction)
        assert float(loss.sum()) == 0.0
        w.grad = None
        loss.sum().backward()
        assert float(w.grad.abs().max()) == 0.0


@pytest.mark.parametrize('dtype', list(DTYPES))
def test_linear_cross_entropy_values_of_ignored_rows_do_not_matter(S, dtype):
    """Infinities and NaN in rows that are ignored: the same bits as zeros there, and a gradient of zero."""
    x, w, t, g = lce_case(50, 40, 200, dtype, 0.4)
    res = []
    for fill in (0.0, float('nan'), float('inf'), -torch.finfo(DTYPES[dtype]).max):
        y = x.clone()
        y[t == IGNORE] = fill
        xg, wg = y.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        loss = S['ops'].linear_cross_entropy(xg, wg, t.cuda())
        loss.backward()
        res.append((loss.detach().clone(), xg.grad, wg.grad))
        assert float(xg.grad.cpu()[t == IGNORE].abs().max()) == 0.0
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(res[0], r))


def test_linear_cross_entropy_unknown_target_is_nan(S):
    x, w, t, g = lce_case(20, 24, 50, 'fp32', 0.0)
    for bad in (50, -1, 1 << 40):
        t2 = t.clone()
        t2[7] = bad
        xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        loss = S['ops'].linear_cross_entropy(xg, wg, t2.cuda(), reduction='none')
        ok = torch.arange(20) != 7
        assert torch.isnan(loss[7]) and torch.isfinite(loss.detach().cpu()[ok]).all()
        loss.sum().backward()
        assert torch.isnan(xg.grad[7]).all() and torch.isfinite(xg.grad.cpu()[ok]).all() and torch.isnan(wg.grad).all()


def test_linear_cross_entropy_large_logits(S):
    """Logits of hundreds: the exponentials do not overflow, a certain target has a loss of 0, an impossible one its distance."""
    w = torch.eye(8, 64)
    x = torch.zeros(3, 64)
    x[:, 2] = 600.0
    t = torch.tensor([2, 5, IGNORE])
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = S['ops'].linear_cross_entropy(xg, wg, t.cuda(), reduction='none')
    assert loss.tolist() == [0.0, 600.0, 0.0]
    loss.sum().backward()
    want = torch.zeros(3, 64)
    want[1, 2], want[1, 5] = 1.0, -1.0
    assert torch.equal(xg.grad.cpu(), want)


@pytest.mark.parametrize('dtype', list(DTYPES))
def test_linear_cross_entropy_words_of_the_lowest_value(S, dtype):
    """Words that their weights rule out, every one the type's lowest value: as if the vocabulary did not have them."""
    x, w, t, g = lce_case(40, 24, 300, dtype, 0.2)
    x = x.abs() + 0.125
    t = torch.where(t == IGNORE, t, t % 250)
    low = w.clone()
    low[250:] = torch.finfo(w.dtype).min
    gout = torch.randn((), generator=g)
    (l, lb), (dx, dxb), (dw, dwb) = lce_reference(x, w[:250], t, gout, 'mean')
    xg, wg = x.cuda().requires_grad_(True), low.cuda().requires_grad_(True)
    loss = S['ops'].linear_cross_entropy(xg, wg, t.cuda())
    within(loss, l, lb)
    loss.backward(gout.cuda())
    within(xg.grad, dx, dxb)
    within(wg.grad[:250], dw, dwb)
    assert float(wg.grad[250:].abs().max()) == 0.0


@pytest.mark.parametrize('dtype', list(DTYPES))
def test_linear_cross_entropy_powers_of_two_of_rows_and_words_cancel(S, dtype):
    """Rows and words of very different sizes whose products are ordinary: a power of two changes no bit of the loss, and moves the
    gradients by itself."""
    x, w, t, _ = lce_case(70, 40, 300, dtype, 0.2)

    def run(x, w):
        x, w = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        loss = S['ops'].linear_cross_entropy(x, w, t.cuda(), ignore_index=IGNORE, reduction='sum')
        loss.backward()
        return loss.detach(), x.grad, w.grad
    loss, dx, dw = run(x, w)
    for up in (30, -50):
        l2, dx2, dw2 = run(x * 2.0 ** up, w * 2.0 ** -up)
        assert torch.equal(loss, l2)
        assert torch.equal(dx * 2.0 ** -up, dx2) and torch.equal(dw * 2.0 ** up, dw2)


def test_linear_cross_entropy_columns_of_many_sizes(S):
    """Within a row values down to 2^-16 of the largest, the words the other way round, so that every column counts alike."""
    x, w, t, g = lce_case(50, 48, 300, 'fp32', 0.0)
    size = 2.0 ** -(torch.arange(48) % 17).float()
    lce_check(S, x * size, w / size, t, g, 'mean')


@pytest.mark.parametrize('dtype', list(DTYPES))
def test_linear_cross_entropy_strides(S, dtype):
    """x as a slice, transposed and broadcast; weight as a slice of columns and at an odd offset; targets int32 and strided."""
    g = torch.Generator().manual_seed(17)
    xb, wb = torch.randn(6, 30, 80, generator=g).to(DTYPES[dtype]), torch.randn(301, 80, generator=g).to(DTYPES[dtype])
    t = torch.randint(0, 300, (30, 6), generator=g)
    views = [(lambda b: b[:, :, 5:69].transpose(0, 1), lambda b: b[1:, 9:73]), (lambda b: b[:, :, 8:72].transpose(0, 1), lambda b: b[:300, 8:72]),
             (lambda b: b[:1, :, :64].expand(6, 30, 64).transpose(0, 1), lambda b: b[:300, :1].expand(300, 64))]
    for xv, wv in views:
        x, w = xv(xb), wv(wb)
        gout = torch.tensor(0.7)
        (l, lb), (dx, dxb), (dw, dwb) = lce_reference(x.reshape(-1, 64), w, t.reshape(-1), gout, 'mean')
        xg, wg = xv(xb.cuda()).detach().requires_grad_(True), wv(wb.cuda()).detach().requires_grad_(True)
        loss = S['ops'].linear_cross_entropy(xg, wg, t.to(torch.int32).cuda())
        within(loss, l, lb)
        gx, gw = torch.autograd.grad(loss, (xg, wg), gout.cuda())
        within(gx.reshape(-1, 64), dx, dxb)
        within(gw, dw, dwb)


def test_linear_cross_entropy_one_gradient_only(S):
    x, w, t, g = lce_case(60, 48, 300, 'bf16', 0.2)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    both = torch.autograd.grad(S['ops'].linear_cross_entropy(xg, wg, t.cuda()), (xg, wg))
    (dx,) = torch.autograd.grad(S['ops'].linear_cross_entropy(xg, w.cuda(), t.cuda()), (xg,))
    (dw,) = torch.autograd.grad(S['ops'].linear_cross_entropy(x.cuda(), wg, t.cuda()), (wg,))
    assert torch.equal(dx, both[0]) and torch.equal(dw, both[1])


def test_linear_cross_entropy_gradient_against_differences(S):
    """The change of the loss along a direction: central differences of a loss in 64 bits at a step whose own errors are small."""
    x, w, t, g = lce_case(12, 20, 40, 'fp32', 0.25)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    gx, gw = torch.autograd.grad(S['ops'].linear_cross_entropy(xg, wg, t.cuda()), (xg, wg))
    ux, uw = torch.randn(x.shape, generator=g).double(), torch.randn(w.shape, generator=g).double()

    def loss(h):
        return lce_reference((x.double() + h * ux), (w.double() + h * uw), t, torch.tensor(1.0), 'mean')[0][0]
    h = 1e-5
    slope = float((loss(h) - loss(-h)) / (2 * h))
    got = float((gx.cpu().double() * ux).sum() + (gw.cpu().double() * uw).sum())
    # differences: h^2 times a third derivative of order (|u| |x|)^3 ~ 1e3 -> 1e-7; gradients: fp32 sums, 1e-5 of them at most
    assert abs(slope - got) < 1e-5 * (float((gx.cpu().double() * ux).abs().sum() + (gw.cpu().double() * uw).abs().sum())) + 1e-6


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('ignored', [0.0, 0.95, 1.0])
@pytest.mark.parametrize('reduction', ['mean', 'none'])
def test_linear_cross_entropy_many_rows_few_words(S, reduction, ignored, dtype):
    """The weight's gradient in parts of the rows, more parts than rows that count among them."""
    x, w, t, g = lce_case(1100, 70, 130, dtype, ignored)
    lce_check(S, x, w, t, g, reduction)


def test_linear_cross_entropy_many_rows_few_words_in_the_arena(S):
    x, w, t, g = lce_case(1500, 36, 150, 'fp32', 0.3)
    p, xg = torch.nn.Parameter(w.cuda()), x.cuda()
    arena = S['optim'].ParamArena([p])
    start = torch.randn(arena.numel, generator=g)
    arena.grad.copy_(start.cuda())
    _, _, (dw, dwb) = lce_reference(x, w, t, torch.tensor(1.0), 'mean')
    S['ops'].linear_cross_entropy(xg, p, t.cuda()).backward()
    before = start[:w.numel()].view_as(w).double()
    within(p.grad, before + dw, dwb + U * (before.abs() + dw.abs() + dwb) * 1.01)


def test_linear_cross_entropy_adds_to_the_arena(S):
    x, w, t, g = lce_case(33, 20, 90, 'fp32', 0.3)
    p = torch.nn.Parameter(w.cuda())
    arena = S['optim'].ParamArena([p])
    start = torch.randn(arena.numel, generator=g)
    arena.grad.copy_(start.cuda())
    _, _, (dw, dwb) = lce_reference(x, w, t, torch.tensor(1.0), 'mean')
    S['ops'].linear_cross_entropy(x.cuda(), p, t.cuda()).backward()
    before = start[:w.numel()].view(w.shape).double()
    within(p.grad, before + dw, dwb + U * (before.abs() + dw.abs() + dwb) * 1.01)


def test_linear_cross_entropy_refusals(S):
    f = S['ops'].linear_cross_entropy
    x, w, t = torch.zeros(4, 6).cuda(), torch.zeros(5, 6).cuda(), torch.zeros(4, dtype=torch.int64).cuda()
    for a, kw, err in [((x.half(), w.half(), t), {}, TypeError), ((x, w.bfloat16(), t), {}, TypeError), ((x, w, t.float()), {}, TypeError),
                       ((x, w[:, :5], t), {}, ValueError), ((x, w, t[:3]), {}, ValueError), ((x, w[:0], t), {}, ValueError),
                       ((x, w, t), dict(reduction='median'), ValueError), ((x[0, 0], w, t), {}, ValueError), ((x, w, None), {}, TypeError)]:
        with pytest.raises(err):
            f(*a, **kw)


# ---- gradient norm and clipping ------------------------------------------------------------------------------------------------
def clip_reference(grads, max_norm, norm_type):
    gs = [t.detach().cpu().double() for t in grads]
    norm = math.sqrt(sum(float(t.square().sum()) for t in gs)) if norm_type == 2 else max([float(t.abs().max()) for t in gs if t.numel()], default=0.0)
    return norm, min(1.0, max_norm / (norm + 1e-6)), gs


def clip_check(S, grads, max_norm, norm_type=2.0, out=None):
    norm, f, gs = clip_reference(grads, max_norm, norm_type)
    got = S['optim'].clip_grads(grads, max_norm, norm_type, out=out)
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - norm) <= norm * 2 * U
    for t, o in zip(gs, grads if out is None else out):
        # the norm rounded, 1e-6 added, the quotient, the product: 4 u and what they compound to
        within(o, t * f, (t * f).abs() * (6 * U + half_eps(o.dtype) * (1 + 6 * U)))


SIZES = [[1], [7, 0, 3], [16384], [16385, 16383, 1], [5, 100000, 33, 2, 70001], [3] * 130, [2048] * 257]


@pytest.mark.parametrize('norm_type', [2.0, math.inf])
@pytest.mark.parametrize('dtype', ['fp32', 'bf16', 'mixed'])
@pytest.mark.parametrize('sizes', SIZES, ids=lambda s: f'{len(s)}x{max(s)}')
def test_clip_grads(S, sizes, dtype, norm_type):
    g = torch.Generator().manual_seed(sum(sizes))
    kinds = [DTYPES[dtype] if dtype != 'mixed' else (torch.float32, torch.bfloat16)[k % 2] for k in range(len(sizes))]
    host = [torch.randn(n, generator=g).to(d) for n, d in zip(sizes, kinds)]
    for max_norm in (0.25, 1e6):
        clip_check(S, [t.cuda() for t in host], max_norm, norm_type)
    grads = [t.cuda() for t in host]
    out = [torch.full_like(t, 9.0, dtype=(torch.float32, torch.bfloat16)[(k // 2) % 2]) for k, t in enumerate(grads)]
    clip_check(S, grads, 0.25, norm_type, out=out)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(grads, host))         # inputs of an `out` call stay


def test_clip_grads_offsets_and_orders(S):
    """Tensors that begin at odd elements (two bytes off a vector), a transposed one, one of zero dimensions."""
    g = torch.Generator().manual_seed(4)
    base = torch.randn(40001, generator=g)
    for dt in (torch.float32, torch.bfloat16):
        b = base.to(dt).cuda()
        grads = [b[1:20000], b[20003:20003 + 60 * 70].view(60, 70).t(), b[30000], b[30001:40001].view(100, 100)]
        keep = b.clone()
        clip_check(S, grads, 0.5)
        for at in (0, 20000, 20001, 20002):
            assert torch.equal(b[at], keep[at])


def test_clip_grads_keeps_the_bits_where_nothing_is_clipped(S):
    t = torch.randn(5000, generator=torch.Generator().manual_seed(2)).cuda()
    before = t.clone()
    S['optim'].clip_grads([t], 1e9)
    assert torch.equal(t, before)
    S['optim'].clip_grads([t], math.inf)
    assert torch.equal(t, before)


def test_clip_grads_values_out_of_the_ordinary(S):
    """Squares beyond fp32's range either way; infinities and NaN as the formula has them."""
    big = torch.full((1000,), 1e30).cuda()
    n = S['optim'].clip_grads([big], 1.0)
    assert abs(float(n) / (1e30 * math.sqrt(1000)) - 1) < 1e-6 and abs(float(big[0]) * math.sqrt(1000) - 1) < 1e-6
    small = torch.full((1000,), 1e-30).cuda()
    assert abs(float(S['optim'].clip_grads([small], 1.0)) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    for norm_type in (2.0, math.inf):
        for at in (0, 16, 999):
            x = torch.ones(1000)
            x[at] = float('inf')
            x = x.cuda()
            assert float(S['optim'].clip_grads([x], 1.0, norm_type)) == math.inf
            assert torch.isnan(x[at]) and float(x[(at + 1) % 1000]) == 0.0
            x = torch.ones(1000)
            x[at] = float('nan')
            x = x.cuda()
            assert math.isnan(float(S['optim'].clip_grads([x], 1.0, norm_type)))
            assert torch.isnan(x).all()
        x, y = torch.ones(1000).cuda(), torch.full((7,), float('nan')).cuda()
        assert math.isnan(float(S['optim'].clip_grads([x, y], math.inf, norm_type))) and torch.isnan(x).all()
        x = torch.randn(1000).cuda()
        y = x.clone()
        assert float(S['optim'].clip_grads([x], math.inf, norm_type)) > 0 and torch.equal(x, y)
    z = torch.zeros(30).cuda()
    assert float(S['optim'].clip_grads([z], 1.0)) == 0.0 and float(z.abs().max()) == 0.0
    assert float(S['optim'].clip_grads([torch.zeros(0).cuda()], 1.0)) == 0.0


def test_clip_grads_same_tensor_twice_counts_once(S):
    t = torch.randn(3000, generator=torch.Generator().manual_seed(8))
    a = t.cuda()
    n = S['optim'].clip_grads([a, a], 0.5)
    b = t.cuda()
    assert float(n) == float(S['optim'].clip_grads([b], 0.5)) and torch.equal(a, b)


def test_clip_grad_norm_over_parameters_and_arena(S):
    g = torch.Generator().manual_seed(6)
    ps = [torch.nn.Parameter(torch.zeros(*s).cuda()) for s in ((30, 7), (11,), (5, 5))]
    gr = [torch.randn(p.shape, generator=g) for p in ps]
    ps[0].grad, ps[2].grad = gr[0].cuda(), gr[2].cuda()
    norm, f, _ = clip_reference([gr[0], gr[2]], 0.1, 2)
    n = S['optim'].clip_grad_norm_(ps, 0.1)
    assert abs(float(n) - norm) <= 2 * U * norm
    for p, t in ((ps[0], gr[0]), (ps[2], gr[2])):
        within(p.grad, t.double() * f, t.double().abs() * f * 8 * U)
    arena = S['optim'].ParamArena(ps)
    adam = S['optim'].FusedAdam(arena, 1e-3)
    for p, t in zip(ps, gr):
        p.grad.copy_(t.cuda())
    norm, f, _ = clip_reference(gr, 0.1, 2)
    n = adam.clip_grad_norm(0.1)
    assert abs(float(n) - norm) <= 2 * U * norm
    for p, t in zip(ps, gr):
        within(p.grad, t.double() * f, t.double().abs() * f * 8 * U)


def test_clip_grads_refusals(S):
    f = S['optim'].clip_grads
    t = torch.zeros(10, 10).cuda()
    for a, kw, err in [(([], 1.0), {}, ValueError), (([t], -1.0), {}, ValueError), (([t], float('nan')), {}, ValueError), (([t], 1.0, 1.0), {}, ValueError),
                       (([t.half()], 1.0), {}, TypeError), (([t[:, :5]], 1.0), {}, ValueError), (([t[0].expand(4, 10)], 1.0), {}, ValueError),
                       (([t, t[2:4]], 1.0), {}, ValueError), (([t], 1.0), dict(out=[]), ValueError), (([t], 1.0), dict(out=[t[:5]]), ValueError),
                       (([t], 1.0), dict(out=[torch.zeros(10, 10).cuda().t()]), ValueError),
                       (([t[:5], t[5:]], 1.0), dict(out=[t[5:], t[:5]]), ValueError)]:
        with pytest.raises(err):
            f(*a, **kw)


# ---- streams, graphs, large tensors, a run of them together ---------------------------------------------------------------------
def text_step(S, x, w, ids, table, target, grads, max_norm=0.5):
    """One pass of each operator with all gradients; tensors of a few hundred rows."""
    y = S['ops'].embedding_sorted(ids, table, scale=3.0)
    (dt,) = torch.autograd.grad(y, (table,), x.detach())
    loss = S['ops'].linear_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, (x, w))
    out = [torch.empty_like(g) for g in grads]
    norm = S['optim'].clip_grads(grads, max_norm, out=out)
    return [y.detach(), dt, loss.detach(), dx, dw, norm] + out


def text_inputs(seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    n, d, v = 300, 72, 1500
    x, w, table = (torch.randn(*s, generator=g).to(dtype).cuda() for s in ((n, d), (v, d), (v, d)))
    ids, target = torch.randint(0, v, (n,), generator=g), torch.randint(0, v, (n,), generator=g)
    target[::7] = IGNORE
    ids[::2] = 0
    return x, w, ids.cuda(), table, target.cuda(), [torch.randn(700, generator=g).cuda(), torch.randn(3, 5, generator=g).to(dtype).cuda()]


@pytest.mark.skipif(EMU, reason='graphs and streams are not modelled')
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_text_operators_in_captured_graphs(S, dtype):
    """Forward and backward of all three captured twice on the same inputs' buffers; replays in turn, with new inputs and eager work
    between them, give the eager results' bits."""
    static = text_inputs(1, DTYPES[dtype])
    live = [t for t in static[:5]] + static[5]

    def leaves():
        x, w, ids, table, target, grads = static
        return x.detach().requires_grad_(True), w.detach().requires_grad_(True), ids, table.detach().requires_grad_(True), target, grads
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        text_step(S, *leaves())
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = text_step(S, *leaves())
        graphs.append((g, out))
    for seed in range(2, 6):
        fresh = text_inputs(seed, DTYPES[dtype])
        want = text_step(S, *[t.requires_grad_(True) if i in (0, 1, 3) else t for i, t in enumerate(fresh)])
        for a, b in zip(live, [t for t in fresh[:5]] + fresh[5]):
            a.copy_(b.detach())
        for g, out in (graphs[seed % 2], graphs[1 - seed % 2]):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.skipif(EMU, reason='graphs and streams are not modelled')
def test_text_operators_on_two_streams_at_once(S):
    ins = [text_inputs(s) for s in (11, 12)]
    for i in ins:
        for k in (0, 1, 3):
            i[k].requires_grad_(True)
    want = [text_step(S, *i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [None, None]
    for rep in range(3):
        for k, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[k] = text_step(S, *ins[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.skipif(EMU, reason='gigabytes')
def test_embedding_sorted_offsets_beyond_32_bits(S):
    entries, dim = (1 << 20) + 40001, 2080                 # 2.26e9 elements
    t = torch.zeros(entries, dim, dtype=torch.bfloat16, device='cuda')
    rows = torch.tensor([0, 5, 1 << 20, entries - 2, entries - 1, entries - 1])
    g = torch.Generator().manual_seed(1)
    vals = torch.randn(5, dim, generator=g).to(torch.bfloat16)
    t[rows[:5].cuda()] = vals.cuda()
    t.requires_grad_(True)
    ids = rows.repeat(40).cuda()
    y = S['ops'].embedding_sorted(ids, t)
    assert torch.equal(y[:5].detach().cpu(), vals) and torch.equal(y[5].detach().cpu(), vals[4])
    (dt,) = torch.autograd.grad(y, (t,), torch.ones_like(y))
    assert torch.equal(dt[rows.cuda()].float().cpu(), torch.tensor([40., 40., 40., 40., 80., 80.])[:, None].expand(6, dim))
    assert float(dt.sum(dtype=torch.float64)) == 240.0 * dim


@pytest.mark.skipif(EMU, reason='gigabytes')
def test_clip_grads_offsets_beyond_32_bits(S):
    n = (1 << 32) + 70003
    t = torch.full((n,), 2.0 ** -10, dtype=torch.bfloat16, device='cuda')
    t[-1] = 8.0
    norm = math.sqrt((n - 1) * 2.0 ** -20 + 64.0)
    got = S['optim'].clip_grads([t], norm / 2)
    assert abs(float(got) - norm) <= 2 * U * norm
    assert float(t[0]) == 2.0 ** -11 and float(t[(1 << 32) + 5]) == 2.0 ** -11 and float(t[-1]) == 4.0
    assert float(t[:-1].max()) == 2.0 ** -11 == float(t[:-1].min())


@pytest.mark.skipif(EMU, reason='gigabytes')
def test_linear_cross_entropy_offsets_beyond_32_bits(S):
    """The most rows there may be, 2.3e9 elements of x: the last rows as they are by themselves, to the bounds."""
    n, d, v = 1 << 21, 1088, 40
    g = torch.Generator().manual_seed(21)
    w = torch.randn(v, d, generator=g) * 0.05
    w = w.to(torch.bfloat16)
    x = torch.randn(512, d, generator=g).to(torch.bfloat16)
    t = torch.randint(0, v, (512,), generator=g)
    xg = x.cuda().repeat(n // 512, 1).requires_grad_(True)
    loss = S['ops'].linear_cross_entropy(xg, w.cuda(), t.cuda().repeat(n // 512), reduction='none')
    (l, lb), (dx, dxb), _ = lce_reference(x, w, t, torch.ones(512), 'none')
    within(loss[-512:], l, lb)
    (gx,) = torch.autograd.grad(loss, (xg,), torch.ones_like(loss))
    within(gx[-512:], dx, dxb)
    within(gx[:512], dx, dxb)
    del xg, gx, loss


def test_linear_cross_entropy_kept_graph_and_one_row(S):
    x, w, t, g = lce_case(40, 24, 100, 'fp32', 0.2)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = S['ops'].linear_cross_entropy(xg, wg, t.cuda())
    a = torch.autograd.grad(loss, (xg, wg), retain_graph=True)
    b = torch.autograd.grad(loss, (xg, wg))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    one = S['ops'].linear_cross_entropy(xg[3], wg, t.cuda()[3], reduction='none')       # a vector and a number
    assert one.shape == () and torch.equal(one.detach(), S['ops'].linear_cross_entropy(xg, wg, t.cuda(), reduction='none')[3].detach())


def test_text_operators_prepare_no_backward_pass_without_grad_mode(S, monkeypatch):
    """Parameters under no_grad: scoring a model keeps nothing for a backward pass that cannot come."""
    from speech2affective_gestures_amd import text
    kept = []
    real = text._lce_workspace
    monkeypatch.setattr(text, '_lce_workspace', lambda lib, a, backward, device: (kept.append(a.keep), real(lib, a, backward, device))[1])
    x, w, t, _ = lce_case(30, 20, 50, 'fp32', 0.1)
    x, w, t = x.cuda(), torch.nn.Parameter(w.cuda()), t.cuda()
    with torch.no_grad():
        a = S['ops'].linear_cross_entropy(x, w, t)
        e = S['ops'].embedding_sorted(t.clamp(min=0), w)
    assert not a.requires_grad and not e.requires_grad
    b = S['ops'].linear_cross_entropy(x, w, t)
    assert b.requires_grad and torch.equal(a, b.detach())
    assert kept == [0, 1]


def test_linear_cross_entropy_changed_weight_is_noticed(S):
    """A weight that is changed between the passes: torch's own error, not gradients of two different weights."""
    x, w, t, g = lce_case(10, 24, 30, 'fp32', 0.0)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = S['ops'].linear_cross_entropy(xg, wg, t.cuda())
    with torch.no_grad():
        wg += 1.0
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_clip_grads_counts_as_a_change(S):
    t = torch.ones(10).cuda()
    before = t._version
    S['optim'].clip_grads([t], 0.1)
    assert t._version > before


def test_a_step_of_a_text_model(S):
    """The operators as they are used: scaled embedding, a layer of the framework's own, cross entropy over the tied table, the norm
    of all gradients in the arena, clipping, Adam -- against the same step in 64 bits."""
    ops, optim = S['ops'], S['optim']
    g = torch.Generator().manual_seed(31)
    v, d, B, T = 700, 64, 5, 34
    table, mix, bias = torch.randn(v, d, generator=g) * 0.3, torch.randn(d, d, generator=g) / 8, torch.randn(d, generator=g) * 0.1
    ids = torch.randint(0, v, (B, T), generator=g)
    ids[torch.rand(B, T, generator=g) < 0.5] = 0
    target = torch.roll(ids, -1, 1).clone()
    target[:, -1] = IGNORE
    target[target == 0] = IGNORE
    E, M, b = (torch.nn.Parameter(t.cuda()) for t in (table, mix, bias))
    arena = optim.ParamArena([E, M, b])
    adam = optim.FusedAdam(arena, lr=1e-2, betas=(0.9, 0.999), eps=1e-2)
    adam.zero_grad()
    h = ops.linear(ops.embedding_sorted(ids.cuda(), E, scale=8.0).view(B * T, d), M, b)
    loss = ops.linear_cross_entropy(h.view(B, T, d), E, target.cuda())
    loss.backward()
    norm = adam.clip_grad_norm(0.5)
    grads = [p.grad.clone() for p in (E, M, b)]
    adam.step()
    Er, Mr, br = (t.double().requires_grad_(True) for t in (table, mix, bias))
    hr = torch.nn.functional.linear(Er[ids.view(-1)] * 8.0, Mr, br)
    lr_ = torch.nn.functional.cross_entropy(hr @ Er.t(), target.view(-1), ignore_index=IGNORE)
    ref = torch.autograd.grad(lr_, (Er, Mr, br))
    nr = math.sqrt(sum(float(t.square().sum()) for t in ref))
    tol = 1e-4                                             # the layer's own, relative to the largest element (tests/test_gpu_ops.py)
    assert abs(float(loss) - float(lr_)) < tol * float(lr_) and abs(float(norm) - nr) < tol * nr and nr > 0.5
    for p, gr, r, start in zip((E, M, b), grads, ref, (table, mix, bias)):
        r = r * min(1.0, 0.5 / (nr + 1e-6))
        err = tol * float(r.abs().max())
        assert float((gr.cpu().double() - r).abs().max()) < err
        # Adam's first step: lr g / (|g| + eps), which moves by lr / eps of what g is off; the moments' bias corrections cancel
        want = start.double() - 1e-2 * r / (r.abs() + 1e-2)
        assert float((p.detach().cpu().double() - want).abs().max()) < 1e-2 / 1e-2 * err + 1e-6


def _by_clones(run):
    """Saved tensors as copies of themselves, the memory of what was saved given to others before the backward pass."""
    held = []

    def pack(t):
        return t.detach().clone()

    def unpack(t):
        held.extend(torch.full((n,), 0x7f, dtype=torch.uint8, device=t.device) for n in sizes for _ in range(3))
        return t.clone()
    sizes = (64, 512, 1024, 4096, 16384, 65536, 262144)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        return run()


def _on_the_host(run):
    with torch.autograd.graph.save_on_cpu():
        return run()


def _by_checkpoint(run):
    from torch.utils.checkpoint import checkpoint
    return checkpoint(run, use_reentrant=False, preserve_rng_state=False)


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('saving', [_by_clones, _on_the_host, _by_checkpoint])
def test_text_operators_read_the_saved_tensors_that_they_are_given(S, saving, dtype):
    """Hooks on saved tensors and checkpointing hand the backward pass other tensors than were saved: the same bits as without them."""
    ops = S['ops']
    for n, d, v in ((40, 24, 100), (130, 64, 300)):                # (64 columns: bf16 words are read where they lie)
        x, w, t, g = lce_case(n, d, v, dtype, 0.2)
        ids = ids_of('padded', n, v, g)
        dy = torch.randn(n, d, generator=g).to(DTYPES[dtype]).cuda()
        xg, wg, tg, ig = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True), t.cuda(), ids.cuda()
        for run, leaves, grad in ((lambda: ops.linear_cross_entropy(xg, wg, tg), (xg, wg), None),
                                  (lambda: ops.linear_cross_entropy(xg, wg, tg, reduction='none').sum(), (xg, wg), None),
                                  (lambda: ops.embedding_sorted(ig, wg, scale=2.0), (wg,), dy)):
            plain = run()
            want = torch.autograd.grad(plain, leaves, grad)
            other = saving(run)
            got = torch.autograd.grad(other, leaves, grad)
            assert torch.equal(other, plain)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_linear_cross_entropy_in_the_arena_under_a_checkpoint(S):
    """The weight of a ParamArena, its gradient added there once though the forward pass runs twice."""
    x, w, t, g = lce_case(40, 24, 100, 'fp32', 0.2)
    grads = []
    for saving in (lambda run: run(), _by_checkpoint):
        xg, wg = x.cuda().requires_grad_(True), torch.nn.Parameter(w.cuda())
        arena = S['optim'].ParamArena([wg])
        arena.grad.fill_(0.5)
        saving(lambda: S['ops'].linear_cross_entropy(xg, wg, t.cuda())).backward()
        grads.append((xg.grad, wg.grad.clone()))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('factor', [float('inf'), float('nan')])
def test_linear_cross_entropy_ignored_rows_stay_out_of_an_infinite_factor(S, factor, dtype):
    """A loss scale that has overflowed: what the factor does not enter is zero, in every way that the results are written."""
    sizes = [(40, 24, 100), (3000, 16, 130)]                        # dW at once, and in parts of the rows that a launch joins
    for n, d, v in sizes[:1] if EMU and dtype == 'bf16' else sizes:
        x, w, t, g = lce_case(n, d, v, dtype, 0.3)
        none = torch.full_like(t, IGNORE)
        for reduction in ('mean', 'sum', 'none'):
            for target, ignored in ((t, t == IGNORE), (none, none == IGNORE)):
                xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
                loss = S['ops'].linear_cross_entropy(xg, wg, target.cuda(), reduction=reduction)
                loss.backward(torch.full_like(loss, factor))
                dx = xg.grad.cpu()
                assert float(dx[ignored].abs().max()) == 0.0
                if not ignored.all():
                    assert not torch.isfinite(dx[~ignored]).any() and not torch.isfinite(wg.grad).any()
                else:
                    assert float(wg.grad.abs().max()) == 0.0


@pytest.mark.parametrize('reduction', ['mean', 'none'])
def test_linear_cross_entropy_words_ruled_out_by_infinities(S, reduction):
    """bf16 words whose every logit is -infinity: the loss and the other words' gradient as if they were not there, a gradient of zero for
    them (fp32 gives NaN, as is documented).  The input's gradient holds 0 times infinity: NaN."""
    for n in (40, 64, 200):
        x, w, t, g = lce_case(n, 24, 300, 'bf16', 0.2)
        x = x.abs() + 0.125
        t = torch.where(t == IGNORE, t, t % 250)
        low = w.clone()
        low[250:] = -float('inf')
        gout = torch.randn(t.shape if reduction == 'none' else (), generator=g)
        (l, lb), _, (dw, dwb) = lce_reference(x, w[:250], t, gout, reduction)
        xg, wg = x.cuda().requires_grad_(True), low.cuda().requires_grad_(True)
        loss = S['ops'].linear_cross_entropy(xg, wg, t.cuda(), reduction=reduction)
        within(loss, l, lb)
        loss.backward(gout.cuda())
        within(wg.grad[:250], dw, dwb)
        assert float(wg.grad[250:].abs().max()) == 0.0
        assert torch.isnan(xg.grad.cpu()[t != IGNORE]).all() and float(xg.grad.cpu()[t == IGNORE].abs().max()) == 0.0


# ---- fp32's precision over whole results ---------------------------------------------------------------------------------------
# The bounds above are worst cases, element by element, which a missing product of two pieces can hide under where sums are long.  Over
# a whole result errors are independent and its norm is what they add up to: a rounding is 0.58 U of its value at most (rms, half a
# step uniformly over a step, a value at the low end of its binade), one for each of the contraction's `steps` instructions; 8 U for
# G's own (its logarithm and exponent) and what the pieces leave.  A pair of pieces that is left out is 1.5e-6 to 3e-6 of the result.
def norm_bound(steps):
    return U * (8 + math.sqrt(steps))


def pieces_of(v, count, kind):
    out, rest = [], v.float()
    for _ in range(count):
        out.append(rest.to(kind).float())
        rest = rest - out[-1]
    return [p.double() for p in out]


NORM_CASES = [(130, 300, 1000), (300, 36, 500), (129, 64, 257), (4100, 800, 700), (1000, 520, 65536), (1500, 700, 20000)]


def norm_error(got, ref):
    return float((got.detach().cpu().double() - ref).norm() / ref.norm())


@pytest.mark.parametrize('case', [pytest.param(c, marks=pytest.mark.skipif(EMU and c[0] * c[2] > 1e6, reason='minutes on the device model'))
                                  for c in NORM_CASES])
def test_linear_cross_entropy_keeps_the_precision_of_fp32(S, case):
    n, d, v = case
    x, w, t, g = lce_case(n, d, v, 'fp32', 0.0)
    gout = torch.randn(n, generator=g)                              # (a factor of 1 would be one piece)
    x64, w64 = x.double(), w.double()
    z = x64 @ w64.t()
    lse = torch.logsumexp(z, 1)
    loss = lse - z[torch.arange(n), t]
    z.sub_(lse[:, None]).exp_()
    z[torch.arange(n), t] -= 1.0
    z.mul_(gout.double()[:, None])
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    out = S['ops'].linear_cross_entropy(xg, wg, t.cuda(), reduction='none')
    out.backward(gout.cuda())
    # a loss is a difference of numbers up to 16: two roundings of half of 2^-20, of a loss of 5 and more on average
    assert norm_error(out, loss) < 2.0 ** -20 / 5
    checked = 0
    for got, a, b, long in ((xg.grad, z, w64, v), (wg.grad, z.t(), x64, n)):
        bound = norm_bound(6 * -(-long // 32))
        if bound < 1.5e-6:                                          # (longer ones would not notice a pair)
            checked += 1
            assert norm_error(got, a @ b) < bound
    assert checked


def test_the_bound_on_fp32s_precision_notices_a_missing_pair_of_pieces():
    """The oracle with one product of two pieces left out, in 64 bits otherwise: beyond the bound of every contraction that is held to it."""
    n, d, v = 130, 300, 1000
    x, w, t, g = lce_case(n, d, v, 'fp32', 0.0)
    G = torch.softmax(x.double() @ w.double().t(), 1)
    G[torch.arange(n), t] -= 1.0
    G = (G * torch.randn(n, generator=g).double()[:, None]).float()
    for a, b in ((G, w), (G.t().contiguous(), x)):
        A, B = pieces_of(a, 3, torch.bfloat16), pieces_of(b, 3, torch.bfloat16)
        ref = a.double() @ b.double()
        pairs = [(0, 2), (0, 1), (1, 1), (1, 0), (0, 0), (2, 0)]
        full = sum(A[i] @ B[j] for i, j in pairs)
        assert norm_error(full, ref) < 2 * U
        for i, j in pairs:
            assert norm_error(full - A[i] @ B[j], ref) > 1.5e-6, (i, j)


# ---- gradients that several streams add to the arena -----------------------------------------------------------------------------
def test_passes_that_add_to_one_gradient_take_turns(S, monkeypatch):
    """Which stream waits for which: the one that adds to a parameter's gradient next for the last one, and none for itself or for
    a captured one (on the host alone)."""
    from speech2affective_gestures_amd import text

    class Stream:
        def __init__(self, handle, capturing=False):
            self.cuda_stream, self.capturing, self.waited = handle, capturing, []

        def wait_stream(self, s):
            self.waited.append(s.cuda_stream)
    a, b, c = Stream(1), Stream(2), Stream(3, True)
    now = [a]
    monkeypatch.setattr(text, '_stream', lambda t: now[0].cuda_stream)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda d=None: now[0])
    monkeypatch.setattr(text, '_capturing', lambda s: s.capturing)
    p = torch.nn.Parameter(torch.zeros(4, 3).cuda())
    q = torch.nn.Parameter(torch.zeros(2).cuda())
    S['optim'].ParamArena([p, q])
    for st in (a, a, b, b, a, c, c, b):
        now[0] = st
        assert text._arena_slot(p) is p.grad
    assert a.waited == [2] and b.waited == [1] and c.waited == []
    now[0] = b
    text._arena_slot(q)                                             # (another parameter: its own turns)
    assert b.waited == [1]


@pytest.mark.skipif(EMU, reason='streams of the device')
def test_two_streams_add_to_one_table_of_the_arena(S):
    """Backward passes of lookups that two streams made of one table, the first one's long: nothing is lost."""
    ops = S['ops']
    g = torch.Generator().manual_seed(5)
    entries, dim, n = 5000, 512, 60000
    table = torch.nn.Parameter(torch.randn(entries, dim, generator=g).cuda())
    arena = S['optim'].ParamArena([table])
    ids = [torch.randint(0, entries, (n,), generator=g).cuda() for _ in range(2)]
    dy = [torch.randint(-2, 3, (n, dim), generator=g).float().cuda() for _ in range(2)]       # (whole numbers: any order, one sum)
    want = torch.zeros(entries, dim, device='cuda')
    for i, d in zip(ids, dy):
        want.index_add_(0, i, d)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        arena.grad.zero_()
        ys = []
        for st, i in zip(streams, ids):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                ys.append(ops.embedding_sorted(i, table))
        torch.autograd.backward(ys, dy)
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        assert torch.equal(table.grad, want)


def test_a_parameter_that_has_taken_turns_can_be_saved(S):
    import io
    p = torch.nn.Parameter(torch.randn(4, 3).cuda())
    S['optim'].ParamArena([p])
    S['ops'].embedding_sorted(torch.tensor([1, 2]).cuda(), p).sum().backward()
    f = io.BytesIO()
    torch.save(p, f)
    f.seek(0)
    assert torch.equal(torch.load(f, weights_only=False), p)        # (bytes made above)
