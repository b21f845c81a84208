"""The adapter operators' kernels against their formulas in 64 bits: sizes that no tile divides, groups of rows, masks, strides, streams, graphs."""
import math

import pytest
import torch
from adapter_operators import (loss_inputs, mask_by_formula, policy_by_formula, preference_by_formula, update_by_formula, update_inputs)
from training_operators import within

from oxibonsai_b200 import training as TR
from oxibonsai_b200.training.counter_dropout import keep_steps, kept

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def run_update(x, base, dy, a, b, scales, ids, want="xab", **kw):
    x, a, b = (t.detach().requires_grad_(k in want) for k, t in zip("xab", (x, a, b)))
    y = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, **kw)
    grads = torch.autograd.grad(y, [t for t in (x, a, b) if t.requires_grad], dy) if want else ()
    return (y.detach(), *grads)


def compare(got, want, names):
    for g, w, b, what in zip(got, *want, names):
        if g.dtype == torch.float16:          # from 65520 on, half a step above its largest value, float16 rounds to infinity
            over, near = w.abs() - b >= 65520, w.abs() + b >= 65520
            assert torch.equal(g[over].double(), torch.sign(w[over]) * float("inf")), what
            g, w, b = g[~near], w[~near], b[~near]
        within(g, w, b, what)


NAMES = ("y", "dx", "da", "db")


def check_update(n, d, out, rank, adapters, dtype, seed=0, **kw):
    args = update_inputs(n, d, out, rank, adapters, dtype, DEV, seed=seed, **kw)
    got = run_update(*args)
    compare(got, update_by_formula(*args), NAMES)
    assert torch.equal(run_update(*args, want="")[0], got[0])           # served: the small batches' grouping, no rank values kept
    return args, got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, out, rank", [(1, 1, 1, 1), (1, 4096, 64, 16), (2, 7, 9, 2), (15, 64, 33, 8), (16, 128, 32, 16), (17, 129, 31, 17), (63, 72, 200, 5), (65, 1001, 515, 31),
                                             (130, 264, 96, 32), (257, 136, 130, 33), (300, 64, 64, 64), (70, 200, 72, 65), (200, 520, 136, 128), (1024, 256, 264, 16),
                                             (1025, 192, 40, 12), (1500, 65, 63, 100), (2100, 8, 8, 64), (40, 5000, 24, 3)])
def test_update_sizes(n, d, out, rank, dtype):
    check_update(n, d, out, rank, 0, dtype, seed=n + d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", ["mixed", "runs"])
@pytest.mark.parametrize("n, adapters, rank", [(1, 3, 4), (16, 1, 16), (33, 40, 8), (255, 2, 5), (256, 7, 16), (257, 7, 16), (600, 64, 20), (1300, 3, 40), (2050, 30, 128),
                                               (1100, 40, 16), (1030, 200, 8)])
def test_update_groups(n, adapters, rank, spread, dtype):
    args, got = check_update(n, 88, 104, rank, adapters, dtype, seed=n, bare=0.2, spread=spread)
    ids = args[6]
    assert torch.equal(got[0][ids < 0], args[1][ids < 0]) and not got[1][ids < 0].any()
    missing = [e for e in range(adapters) if not (ids == e).any()]
    assert not got[2][missing].any() and not got[3][missing].any()
    again = run_update(*args[:6], ids.int())
    assert all(torch.equal(p, q) for p, q in zip(got, again))


# from 1024 rows and 2^24 results on the two products are kernels of their own: here forward, backward, both; widths that no block divides
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, out, rank, adapters", [(1100, 72, 15360, 16, 0), (1100, 15360, 72, 16, 0), (2050, 8200, 8192, 8, 0), (1029, 65, 16413, 5, 0), (1029, 16413, 65, 3, 0),
                                                       (1030, 64, 16400, 32, 3), (1030, 16400, 64, 24, 3), (1040, 16392, 16384, 8, 70), (1040, 64, 16384, 64, 2),
                                                       (1025, 16384, 8, 100, 40), (1025, 8, 16400, 128, 40), (1024, 16384, 16, 128, 1), (1030, 24, 16392, 16, 70)])
def test_update_in_two_products(n, d, out, rank, adapters, dtype):
    args, got = check_update(n, d, out, rank, adapters, dtype, seed=n + rank, bare=0.1, spread="mixed" if n % 2 else "runs")
    if adapters:
        ids = args[6]
        assert torch.equal(got[0][ids < 0], args[1][ids < 0]) and not got[1][ids < 0].any()
        wrong = ids.clone()
        wrong[[5, n - 1]] = adapters
        bad = run_update(*args[:6], wrong)
        others = wrong != adapters
        assert bad[0][~others].isnan().all() and bad[1][~others].isnan().all()
        assert torch.equal(bad[0][others], got[0][others]) and torch.equal(bad[1][others], got[1][others])
    elif n * max(d, out) < 2 ** 25:
        args[0][7, 3], args[2][9, 1] = float("nan"), float("inf")
        odd = run_update(*args)
        rows = torch.arange(n, device=DEV)
        assert torch.equal(odd[0][rows != 7], got[0][rows != 7]) and torch.equal(odd[1][rows != 9], got[1][rows != 9])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adapters", [0, 3])
def test_update_in_two_products_with_dropout_in_place_and_alone(adapters, dtype):
    n, d, out = 1100, 15360, 15400
    args = update_inputs(n, d, out, 8, adapters, dtype, DEV, seed=2, bare=0.1)
    seed, steps = 77, keep_steps(0.3)
    keep = kept(n, d, steps, seed).to(DEV)
    got = run_update(*args, dropout=0.3, seed=seed)
    compare(got, update_by_formula(*args, keep=keep, share=65536 / steps), NAMES)
    for want in ("x", "a", "b", "xb"):
        part = run_update(*args, want=want, dropout=0.3, seed=torch.tensor(seed, device=DEV))
        assert all(torch.equal(g, dict(zip("yxab", got))[k]) for g, k in zip(part, "y" + want)), want
    x, base, _, a, b, scales, ids = args
    out_of = base.clone()
    plain = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales)
    assert torch.equal(TR.low_rank_update(x, a, b, base=out_of, ids=ids, scale=scales, out=out_of), plain)
    bare = TR.low_rank_update(x, a, b, ids=ids, scale=scales)
    within(bare, *(t[0] for t in update_by_formula(x, None, args[2], a, b, scales, ids)), "without a base")


# rows at odd addresses, which other threads copy than those that drop them: both products in two kernels, tiles of 64 rows and of 16
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adapters, rank", [(0, 16), (3, 30), (60, 8)])
def test_update_in_two_products_with_dropout_at_odd_addresses(adapters, rank, dtype):
    n, d, out = 1101, 15361, 15401
    args = update_inputs(n, d, out, rank, adapters, dtype, DEV, seed=4, bare=0.1)
    seed, steps = 78, keep_steps(0.3)
    keep = kept(n, d, steps, seed).to(DEV)
    got = run_update(*args, dropout=0.3, seed=seed)
    compare(got, update_by_formula(*args, keep=keep, share=65536 / steps), NAMES)
    again = run_update(*args, dropout=0.3, seed=seed)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 300])
def test_update_rows_alone_and_beside_others(n, dtype):
    """Rows of one adapter have the same bits wherever the others lie; rows without one are left as they are; wrong ids stay with their rows."""
    x, base, dy, a, b, scales, ids = update_inputs(n, 72, 56, 6, 4, dtype, DEV, seed=3, bare=0.2)
    got = run_update(x, base, dy, a, b, scales, ids)
    turn = torch.randperm(n, device=DEV)
    moved = run_update(x[turn], base[turn], dy[turn], a, b, scales, ids[turn])
    assert torch.equal(moved[0], got[0][turn]) and torch.equal(moved[1], got[1][turn])
    wrong = ids.clone()
    wrong[2] = 4
    bad = run_update(x, base, dy, a, b, scales, wrong)
    others = torch.arange(n, device=DEV) != 2
    assert bad[0][2].isnan().all() and bad[1][2].isnan().all() and torch.equal(bad[0][others], got[0][others]) and torch.equal(bad[1][others], got[1][others])
    compare(bad[2:], [t[2:] for t in update_by_formula(x[others], base[others], dy[others], a, b, scales, ids[others])], NAMES[2:])
    for value in (-1, -2 ** 31, 4, 2 ** 31 - 1):
        all_same = run_update(x, base, dy, a, b, scales, torch.full_like(ids, value))
        assert (torch.equal(all_same[0], base) if value < 0 else all_same[0].isnan().all()) and not all_same[2].any() and not all_same[3].any()
    far = torch.full_like(ids, 2 ** 40)
    assert run_update(x, base, dy, a, b, scales, far)[0].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_update_values_that_are_not_finite_stay_in_their_rows(dtype):
    x, base, dy, a, b, scales, ids = update_inputs(90, 80, 40, 5, 3, dtype, DEV, seed=6, bare=0.2)
    want = run_update(x, base, dy, a, b, scales, ids)
    x2, row = x.clone(), int((ids == 1).nonzero()[0])
    x2[row, 3] = float("inf")
    x2[int((ids < 0).nonzero()[0])] = float("nan")
    got = run_update(x2, base, dy, a, b, scales, ids)
    keep = torch.arange(90, device=DEV) != row
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1], want[1])
    assert not got[0][row].isfinite().any()
    alone = TR.low_rank_update(x2[row:row + 1].abs(), torch.ones_like(a[1:2]), torch.ones_like(b[1:2]))
    assert torch.isposinf(alone).all() if dtype != torch.float32 else not alone.isfinite().any()
    assert torch.equal(got[2][[0, 2]], want[2][[0, 2]]) and torch.equal(got[3][[0, 2]], want[3][[0, 2]])


@pytest.mark.parametrize("dtype", TYPES)
def test_update_exact_sums(dtype):
    """Whole numbers whose sums fit 22 bits come out as they are: no rank value is rounded to 16 bits on the way."""
    g = torch.Generator().manual_seed(5)
    whole = lambda top, *shape: torch.randint(-top, top + 1, shape, generator=g).to(DEV, dtype)  # noqa: E731
    for n, adapters in ((200, 0), (1100, 2)):
        e = max(1, adapters)
        x, a, b, dy = whole(15, n, 512), whole(15, e, 8, 512), whole(1, e, 24, 8), whole(15, n, 24)
        ids = torch.randint(0, e, (n,), generator=g).to(DEV) if adapters else None
        (y, dx, da, db), _ = update_by_formula(x, None, dy, a, b, torch.ones(e, device=DEV), ids)
        got = run_update(x, None, dy, a, b, 1.0, ids)
        assert float(y.abs().max()) < 2 ** 22
        for have, want in zip(got, (y, dx, da, db)):
            assert torch.equal(have, want.to(dtype)) if float(want.abs().max()) < 2 ** 22 else True
        assert torch.equal(got[0], y.to(dtype)) and torch.equal(got[1], dx.to(dtype))


def test_update_f32_keeps_its_bits():
    """Operands of 24 bits: two TF32 parts of each leave 2^-20 of a single product's magnitude, one part would leave 2^-11."""
    g = torch.Generator().manual_seed(9)
    for n in (3, 1100):
        x, a, b = torch.rand(n, 4, generator=g) + 1, torch.rand(1, 1, 4, generator=g) + 1, torch.rand(1, 16, 1, generator=g) + 1
        dy = torch.rand(n, 16, generator=g) + 1
        args = [t.to(DEV) for t in (x, dy, a, b)]
        got = run_update(args[0], None, args[1], args[2], args[3], 1.0, None)
        want, _ = update_by_formula(args[0], None, args[1], args[2], args[3], torch.ones(1, device=DEV), None)
        for have, exact in zip(got, want):
            assert float(((have.double() - exact) / exact).abs().max()) < 2.0 ** -19


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, out, adapters, p", [(5, 40, 24, 0, 0.5), (70, 37, 50, 3, 0.25), (1100, 136, 72, 0, 0.1), (300, 9, 130, 2, 0.9), (20, 64, 64, 2, 1.0)])
def test_update_dropout(n, d, out, adapters, p, dtype):
    args = update_inputs(n, d, out, 7, adapters, dtype, DEV, seed=n, bare=0.1)
    seed, steps = 2 ** 40 + n, keep_steps(p)
    keep, share = kept(n, d, steps, seed).to(DEV), 65536 / steps if steps else 0.0
    got = run_update(*args, dropout=p, seed=seed)
    compare(got, update_by_formula(*args, keep=keep, share=share), NAMES)
    if adapters == 0:
        x = args[0].clone()
        x[~keep] = float("nan")             # what is dropped reaches nothing
        same = run_update(x, *args[1:], dropout=p, seed=torch.tensor(seed, device=DEV))
        assert all(torch.equal(g, s) for g, s in zip(got, same))


@pytest.mark.parametrize("dtype", TYPES)
def test_update_strides_orders_and_out(dtype):
    x, base, dy, a, b, scales, ids = update_inputs(40, 48, 24, 8, 3, dtype, DEV, seed=1, bare=0.2)
    want = run_update(x, base, dy, a, b, scales, ids)
    wide = torch.randn(40, 61, device=DEV).to(dtype)
    wide[:, 3:51] = x
    tall = torch.randn(40, 3, 24, device=DEV).to(dtype)
    tall[:, 1] = base
    same = [(wide[:, 3:51], base, dy, a, b), (x.T.contiguous().T, tall[:, 1], dy, a, b), (x, base.T.contiguous().T, dy.T.contiguous().T, a, b),
            (x, base, dy, a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(0, 1).contiguous().transpose(0, 1))]
    for case in same:
        compare(run_update(*case, scales, ids), update_by_formula(*case, scales, ids), NAMES)
    spread = ids.repeat_interleave(2)[::2]
    assert all(torch.equal(g, w) for g, w in zip(run_update(x, base, dy, a, b, scales, spread), want))
    row = x[:1].expand(40, 48)
    compare(run_update(row, base[:1].expand(40, 24), dy[:1].expand(40, 24), a, b, scales, ids),
            update_by_formula(row, base[:1].expand(40, 24), dy[:1].expand(40, 24), a, b, scales, ids), NAMES)
    shaped = run_update(x.view(4, 10, 48), base.view(4, 10, 24), dy.view(4, 10, 24), a, b, scales, ids.view(4, 10))
    assert torch.equal(shaped[0].flatten(0, 1), want[0]) and torch.equal(shaped[1].flatten(0, 1), want[1])
    for at in (0, 3, 24):
        block = torch.randn(40, 72, device=DEV).to(dtype)
        block[:, at:at + 24] = base
        whole, out = block.clone(), block[:, at:at + 24]
        got = TR.low_rank_update(x, a, b, base=out, ids=ids, scale=scales, out=out)
        whole[:, at:at + 24] = want[0]
        assert got is out and torch.equal(block, whole)              # in place, and nothing beside it
    fresh = torch.full((40, 24), float("nan"), device=DEV, dtype=dtype)
    assert torch.equal(TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, out=fresh), want[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, out, rank", [(3, 256, 192, 8), (3, 256, 192, 5), (300, 256, 192, 8), (1100, 15360, 15488, 8), (1100, 15360, 15360, 4), (1100, 128, 15360, 16),
                                             (1100, 15360, 128, 16), (1100, 15360, 15360, 24), (1100, 15360, 15360, 40)])
def test_update_reads_its_own_factors(n, d, out, rank, dtype):
    """NaN before and behind the factors, the rows and the base: nothing of it is read into a result."""
    x, base, dy, a, b, scales, _ = update_inputs(n, d, out, rank, 0, dtype, DEV, seed=n)
    want = run_update(x, base, dy, a, b, scales, None)

    def fenced(t):
        room = torch.full((t.numel() + 2 ** 21,), float("nan"), dtype=dtype, device=DEV)
        room[2 ** 20:2 ** 20 + t.numel()] = t.flatten()
        return room[2 ** 20:2 ** 20 + t.numel()].view(t.shape)

    got = run_update(*(fenced(t) for t in (x, base, dy, a, b)), scales, None)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adapters", [0, 3])
def test_update_wanted_gradients(adapters, dtype):
    args = update_inputs(150, 72, 40, 6, adapters, dtype, DEV, seed=4, bare=0.1)
    full = dict(zip("yxab", run_update(*args, dropout=0.2, seed=5)))
    for want in ("x", "a", "b", "xa", "xb", "ab"):
        got = run_update(*args, want=want, dropout=0.2, seed=5)
        assert all(torch.equal(g, full[k]) for g, k in zip(got, "y" + want)), want
    x, base, dy, a, b, scales, ids = args
    base = base.clone().requires_grad_()
    y = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales)
    assert torch.equal(torch.autograd.grad(y, base, dy, retain_graph=True)[0], dy)
    up, = torch.autograd.grad(y.sum(), base)
    assert torch.equal(up, torch.ones_like(base))


def test_update_gradient_by_differences():
    x, base, dy, a, b, scales, ids = update_inputs(40, 32, 24, 4, 2, torch.float32, DEV, seed=8)
    _, *grads = run_update(x, base, dy, a, b, scales, ids)
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        given = [x, a, b]
        way = torch.randn(given[i].shape, generator=g).to(DEV)
        ends = []
        for side in (1, -1):
            args = list(given)
            args[i] = given[i] + side * 0.5 * way
            ends.append(float((TR.low_rank_update(args[0], args[1], args[2], ids=ids, scale=scales).double() * dy).sum()))
        # linear in each: what is left is rounding, 2^-20 of some thousand products of order 1
        assert abs(ends[0] - ends[1] - float((grad.double() * way).sum())) <= 2.0 ** -20 * 40 * 32 * 24


def test_rows_that_are_grouped_without_a_plan():
    from oxibonsai_b200.ops import train_ops
    assert train_ops._LR_SELF_ROWS == train_ops._lib().bonsai_lr_self_rows()


def test_update_no_rows():
    x, base, dy, a, b, scales, ids = update_inputs(4, 16, 8, 2, 3, torch.float32, DEV)
    got = run_update(x[:0], base[:0], dy[:0], a, b, scales, ids[:0])
    assert got[0].shape == (0, 8) and got[1].shape == (0, 16) and not got[2].any() and not got[3].any() and got[2].shape == a.shape


def test_update_streams_and_graphs():
    x, base, dy, a, b, scales, ids = update_inputs(300, 136, 72, 8, 5, torch.bfloat16, DEV, seed=2, bare=0.1)
    seed = torch.tensor(11, device=DEV)
    want = run_update(x, base, dy, a, b, scales, ids, dropout=0.3, seed=11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_update(x, base, dy, a, b, scales, ids, dropout=0.3, seed=seed)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    del got
    sx, sids = x.clone().requires_grad_(), ids.clone()
    sa, sb = a.clone().requires_grad_(), b.clone().requires_grad_()

    def call():
        y = TR.low_rank_update(sx, sa, sb, base=base, ids=sids, scale=scales, dropout=0.3, seed=seed)
        return (y.detach(), *torch.autograd.grad(y, (sx, sa, sb), dy))

    graphs = []
    for _ in range(2):                              # two graphs that may run at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = call()
        graphs.append((graph, held))
    for k in (11, 12):
        seed.fill_(k)
        sids.copy_(ids.roll(k - 11))
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, (graph, _) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want = run_update(x, base, dy, a, b, scales, ids.roll(k - 11), dropout=0.3, seed=k)
        for _, held in graphs:
            assert all(torch.equal(g, w) for g, w in zip(held, want))


@pytest.mark.parametrize("n", [1, 7, 256, 300])
def test_a_bank_in_a_graph(n):
    """Served rows captured and replayed with other rows, ids and adapters, in place; beside an eager call on another stream."""
    x, base, _, a, b, scales, ids = update_inputs(n, 264, 136, 12, 5, torch.float16, DEV, seed=n, bare=0.2)
    bank = TR.AdapterBank(264, 136, rank=12, count=5, dtype=torch.float16, device=DEV)
    bank.a.copy_(a), bank.b.copy_(b), bank.scales.copy_(scales)
    sx, sbase, sids = x.clone(), base.clone(), ids.clone()
    bank(sx, sbase, sids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = bank(sx, sbase, sids)
        bank(sx, y, sids, out=y)                     # a second time on top
    other = torch.cuda.Stream()
    for k in range(3):
        sids.copy_(ids.roll(k))
        sx.copy_(x.roll(k, 1))
        bank.a.copy_(a.roll(k, 0))
        other.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(other):
            z = bank(sx, sbase, sids)
            z = bank(sx, z, sids)
        torch.cuda.synchronize()
        assert torch.equal(y, z)
        want, bound = update_by_formula(sx, sbase, base, bank.a, bank.b, scales, sids)
        within(bank(sx, sbase, sids), want[0], bound[0], "y")


def test_update_places_past_32_bits():
    """Rows whose places in x, base and the result pass 2^31 values."""
    n, cols = 70000, 32768
    base = torch.zeros(n, cols, dtype=torch.bfloat16, device=DEV)
    base[-1] = 1
    x, a, b = torch.randn(n, 8, device=DEV).bfloat16(), torch.randn(8, 8, device=DEV).bfloat16(), torch.randn(cols, 8, device=DEV).bfloat16()
    y = TR.low_rank_update(x, a, b, base=base, out=base)
    want = (x[-3:].double() @ a.double().T) @ b.double().T
    want[-1] += 1
    assert float((y[-3:].double() - want).abs().max()) <= float(want.abs().max()) * 2.0 ** -8
    dy = torch.zeros(n, 8, dtype=torch.bfloat16, device=DEV)
    dy[-3:] = torch.randn(3, 8, device=DEV)
    down, up = b.T.contiguous().requires_grad_(), a.requires_grad_()         # cols to 8
    y.requires_grad_()
    z = TR.low_rank_update(y, down, up)
    dx, da, db = torch.autograd.grad(z, (y, down, up), dy)
    args = y.detach()[-3:], None, dy[-3:], down.detach()[None], up.detach()[None], torch.ones(1, device=DEV), None
    want, bound = update_by_formula(*args)
    for got, w, e, what in zip((z.detach()[-3:], dx[-3:], da[None], db[None]), want, bound, NAMES):
        within(got, w, e, what)
    assert not dx[:-3].any()


def test_update_refusals_on_the_gpu():
    x, base, dy, a, b, scales, ids = update_inputs(6, 8, 5, 3, 4, torch.float32, DEV)
    ok = dict(x=x, a=a, b=b, base=base, ids=ids, scale=scales)
    for change in (dict(ids=ids.cpu()), dict(base=base.cpu()), dict(scale=scales.cpu()), dict(dropout=0.5, seed=torch.tensor(1)), dict(out=base.cpu())):
        with pytest.raises(ValueError):
            TR.low_rank_update(**{**ok, **change})
    with pytest.raises(TypeError):
        TR.low_rank_update(x.double(), a.double(), b.double(), ids=ids)
    z = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(TR.low_rank_update(**{**ok, "x": z}).sum(), z, create_graph=True)


# ---- dropout -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", [(1, 1), (1, 8), (3, 7), (9, 33), (257, 64), (1000, 1001), (70000, 8), (5, 40000), (300, 4096)])
def test_dropout(n, d, dtype):
    g = torch.Generator().manual_seed(n + d)
    x, up = torch.randn(n, d, generator=g).to(dtype), torch.randn(n, d, generator=g).to(dtype)
    for p, seed in ((0.1, 3), (0.75, 2 ** 64 - 5)):
        want = TR.dropout(x, p, seed=seed)
        dx = x.to(DEV).requires_grad_()
        got = TR.dropout(dx, p, seed=seed)
        assert torch.equal(got.detach().cpu(), want)
        assert torch.equal(torch.autograd.grad(got, dx, up.to(DEV))[0].cpu(), TR.dropout(up, p, seed=seed))
    places = [(n - 1, d - 1), (0, 0), (n // 2, d // 2)]
    ones = TR.dropout(torch.ones(n, d, device=DEV), 0.5, seed=9)
    assert torch.equal(torch.stack([ones[r, c] != 0 for r, c in places]).cpu(), mask_by_formula(places, 0.5, 9))


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_strides_and_ends(dtype):
    x = torch.randn(60, 48, device=DEV).to(dtype)
    want = TR.dropout(x, 0.4, seed=5)
    wide = torch.full((60, 61), float("nan"), device=DEV, dtype=dtype)
    for at in (0, 3, 8):
        wide[:, at:at + 48] = x
        assert torch.equal(TR.dropout(wide[:, at:at + 48], 0.4, seed=5), want)
    assert torch.equal(TR.dropout(x.T.contiguous().T, 0.4, seed=5), want)
    assert torch.equal(TR.dropout(x.view(3, 20, 48), 0.4, seed=5).view(60, 48), want)
    assert torch.equal(TR.dropout(x[:1].expand(60, 48), 0.4, seed=5), TR.dropout(x[:1].expand(60, 48).contiguous(), 0.4, seed=5))
    assert torch.equal(TR.dropout(x[0], 0.4, seed=5), want[0])
    gone = torch.full_like(x, float("inf"))
    assert not TR.dropout(gone, 1.0, seed=1).any() and TR.dropout(x, 0.0) is x
    bits = TR.dropout(gone, 0.5, seed=1)
    assert ((bits == 0) | bits.isinf()).all() and (bits == 0).any()
    y = x.clone().requires_grad_()
    twice, = torch.autograd.grad(TR.dropout(y, 0.5, seed=2).float().square().sum(), y, create_graph=True)
    assert torch.autograd.grad(twice.float().sum(), y)[0].max() == 8.0


def test_dropout_seeds_streams_and_graphs():
    x = torch.randn(333, 520, device=DEV)
    seed = torch.tensor(1, device=DEV)
    graph = torch.cuda.CUDAGraph()
    TR.dropout(x, 0.3, seed=seed)
    with torch.cuda.graph(graph):
        y = TR.dropout(x, 0.3, seed=seed)
    for k in (1, 5, -7):
        seed.fill_(k)
        graph.replay()
        assert torch.equal(y, TR.dropout(x, 0.3, seed=k & 2 ** 64 - 1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = TR.dropout(x, 0.3, seed=77)
    side.synchronize()
    assert torch.equal(z, TR.dropout(x, 0.3, seed=77))
    held = torch.randn(4, 8, device=DEV, requires_grad=True)
    out = TR.dropout(held, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    for bad in (torch.tensor(1), torch.tensor([1.0], device=DEV)):
        with pytest.raises(ValueError):
            TR.dropout(x, 0.3, seed=bad)
    assert abs(float((TR.dropout(torch.ones(4096, 4096, device=DEV), 0.3, seed=4) != 0).double().mean()) - 0.7) < 6 * (0.21 / 2 ** 24) ** 0.5


def test_dropout_places_past_32_bits():
    x = torch.ones(70000, 32768, dtype=torch.float16, device=DEV)
    y = TR.dropout(x, 0.5, seed=3)
    places = [(69999, c) for c in range(32760, 32768)] + [(65536, c) for c in range(16)]
    assert torch.equal(torch.stack([y[r, c] == 2 for r, c in places]).cpu(), mask_by_formula(places, 0.5, 3))


# ---- losses ----------------------------------------------------------------------------------------------------------------------------
SIZES = [(2, 1), (2, 130), (6, 7), (10, 511), (4, 512), (34, 2048), (2, 2049), (8, 9001), (600, 12)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, length", SIZES)
def test_preference_sizes(rows, length, dtype):
    for k, (kind, smoothing, average, reduction) in enumerate([("sigmoid", 0.0, False, "mean"), ("sigmoid", 0.15, True, "none"), ("hinge", 0.0, False, "sum"),
                                                               ("ipo", 0.0, True, "mean")]):
        logps, _, ref, mask, _ = loss_inputs(rows, length, dtype, DEV, seed=length + k)
        mask[0] = False
        up = torch.rand(rows // 2, device=DEV) * 1000 if reduction == "none" else torch.tensor(500.0, device=DEV)
        want = preference_by_formula(logps, ref, mask, 0.3, kind, smoothing, average, reduction, up)
        logps[~mask], ref[~mask] = float("nan"), float("inf")
        logps.requires_grad_()
        got = TR.preference_loss(logps, ref, mask, beta=0.3, kind=kind, label_smoothing=smoothing, average=average, reduction=reduction)
        grad, = torch.autograd.grad(got.loss, logps, up)
        assert got.loss.dtype == torch.float32 and grad.dtype == dtype and not grad[~mask].any()
        compare((*(t.detach() for t in got), grad), want, ("loss", "chosen", "rejected", "gradient"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, length", SIZES)
def test_policy_sizes(rows, length, dtype):
    for k, (reduction, per_token, weight) in enumerate([("tokens", True, 0.1), ("sequences", False, 0.0), ("sum", False, 0.2), ("none", True, 0.05)]):
        logps, old, ref, mask, gain = loss_inputs(rows, length, dtype, DEV, seed=length + k)
        mask[0] = False
        gain = gain if per_token else gain[:, 0]
        up = torch.rand(rows, length, device=DEV) if reduction == "none" else torch.tensor(float(rows * length), device=DEV)
        want = policy_by_formula(logps, old, gain, mask, ref, (0.2, 0.3), weight, reduction, up)
        logps[~mask], old[~mask], ref[~mask] = float("nan"), float("inf"), -1e30 if dtype != torch.float16 else -6e4
        logps.requires_grad_()
        got = TR.policy_loss(logps, old, gain, mask=mask, ref_logps=ref, clip=(0.2, 0.3), kl_weight=weight, reduction=reduction)
        grad, = torch.autograd.grad(got.loss, logps, up)
        assert got.loss.dtype == torch.float32 and grad.dtype == dtype and not grad[~mask].any()
        compare((*(t.detach() for t in got), grad), want, ("loss", "kl", "clipped", "gradient"))


@pytest.mark.parametrize("dtype", TYPES)
def test_losses_without_parts(dtype):
    logps, old, ref, mask, gain = loss_inputs(6, 40, dtype, DEV)
    logps.requires_grad_()
    r = TR.policy_loss(logps, None, gain, clip=(1.0, float("inf")))
    want = policy_by_formula(logps.detach(), None, gain, None, None, (1.0, 1e9), 0.0)
    compare((r.loss.detach(), r.kl, r.clipped, torch.autograd.grad(r.loss, logps)[0]), want, ("loss", "kl", "clipped", "gradient"))
    r = TR.preference_loss(logps, None, beta=0.2)
    want = preference_by_formula(logps.detach(), None, None, 0.2, "sigmoid")
    compare((*(t.detach() for t in r), torch.autograd.grad(r.loss, logps)[0]), want, ("loss", "chosen", "rejected", "gradient"))
    nothing = torch.zeros_like(mask)
    for reduction in ("tokens", "sequences"):
        r = TR.policy_loss(logps, old, gain, mask=nothing, reduction=reduction)
        assert r.loss.isnan() and r.clipped.isnan() and not torch.autograd.grad(r.loss, logps)[0].any()
    r = TR.preference_loss(logps, ref, nothing)
    assert abs(float(r.loss.detach()) - 0.6931472) < 1e-6 and not torch.autograd.grad(r.loss, logps)[0].any()
    with torch.no_grad():
        assert not TR.policy_loss(logps, old, gain).loss.requires_grad and not TR.preference_loss(logps, ref).loss.requires_grad


@pytest.mark.parametrize("shape", [(0, 5), (4, 0)])
def test_losses_of_nothing(shape):
    logps = torch.zeros(shape, device=DEV, requires_grad=True)
    for reduction in ("tokens", "sequences", "sum", "none"):
        got = TR.policy_loss(logps, None, torch.zeros(shape[0], device=DEV), ref_logps=torch.zeros(shape, device=DEV), kl_weight=0.1, reduction=reduction)
        assert all(t.device.type == "cuda" for t in got) and got.kl.isnan() and got.clipped.isnan()
        assert got.loss.shape == (shape if reduction == "none" else ())
        assert (got.loss == 0).all() if reduction in ("sum", "none") else got.loss.isnan()
        assert torch.autograd.grad(got.loss.sum(), logps)[0].shape == shape
    got = TR.preference_loss(logps, torch.zeros(shape, device=DEV), reduction="none")
    assert all(t.device.type == "cuda" and t.shape == (shape[0] // 2,) for t in got)
    torch.testing.assert_close(got.loss.cpu(), torch.full((shape[0] // 2,), math.log(2.0)))
    assert torch.autograd.grad(got.loss.sum(), logps)[0].shape == shape


def test_losses_at_their_borders():
    """Ratios next to the clip's borders, gains of zero with infinite ratios, margins that overflow an exponential."""
    l = torch.tensor([[1.2, 1.3, 0.8, 0.7, 1.0]], device=DEV).log()
    steps = torch.tensor([0, 1, -1], device=DEV, dtype=torch.int32)
    logps = (l.view(torch.int32) + steps[:, None]).view(torch.float32)                 # and the neighbours of each
    old = torch.zeros_like(logps)
    for sign in (1.0, -1.0):
        gain = torch.full((3,), sign, device=DEV)
        want = policy_by_formula(logps, old, gain, None, None, (0.2, 0.3), 0.0, "none")
        x = logps.clone().requires_grad_()
        got = TR.policy_loss(x, old, gain, clip=(0.2, 0.3), reduction="none")
        grad, = torch.autograd.grad(got.loss, x, torch.ones_like(x))
        compare((got.loss.detach(), got.kl, got.clipped, grad), want, ("loss", "kl", "clipped", "gradient"))
    x = torch.tensor([[200.0, 200.0, 200.0, -200.0]], device=DEV, requires_grad=True)
    got = TR.policy_loss(x, torch.zeros_like(x), torch.tensor([[0.0, 1.0, -1.0, -1.0]], device=DEV), reduction="none")
    grad, = torch.autograd.grad(got.loss, x, torch.ones_like(x))
    assert got.loss.tolist() == [[0.0, pytest.approx(-1.2), float("inf"), pytest.approx(0.8)]] and grad.tolist() == [[0.0, 0.0, float("inf"), 0.0]]
    x = torch.tensor([[5000.0], [-5000.0], [0.0], [0.0]], device=DEV, requires_grad=True)
    got = TR.preference_loss(x, None, beta=1.0, reduction="none")
    grad, = torch.autograd.grad(got.loss, x, torch.ones(2, device=DEV))
    assert got.loss.tolist() == [0.0, 5000.0] and grad.flatten().tolist() == [0.0, -1.0, 0.0, 1.0]
    up = torch.tensor([float("inf"), 1.0], device=DEV)
    mask = torch.tensor([[True, False]] * 4, device=DEV)
    x = torch.randn(4, 2, device=DEV, requires_grad=True)
    grad, = torch.autograd.grad(TR.preference_loss(x, None, mask, reduction="none").loss, x, up)
    assert grad[[0, 2], 0].isinf().all() and grad[[1, 3], 0].isfinite().all() and not grad[:, 1].any()


def test_losses_strides_streams_and_graphs():
    logps, old, ref, mask, gain = loss_inputs(8, 100, torch.float32, DEV, seed=3)
    want = TR.policy_loss(logps, old, gain, mask=mask, ref_logps=ref, kl_weight=0.1)
    pairs = TR.preference_loss(logps, ref, mask)
    wide = torch.full((8, 103), float("nan"), device=DEV)
    wide[:, 2:102] = logps
    flags = torch.zeros(8, 105, dtype=torch.bool, device=DEV)
    flags[:, 5:] = mask
    got = TR.policy_loss(wide[:, 2:102], old.T.contiguous().T, gain, mask=flags[:, 5:], ref_logps=ref, kl_weight=0.1)
    assert all(abs(float(a) - float(b)) <= 1e-6 for a, b in zip(got, want))
    got = TR.preference_loss(wide[:, 2:102], ref, flags[:, 5:])
    assert all(torch.allclose(a, b, rtol=1e-6) for a, b in zip(got, pairs))
    one = TR.policy_loss(logps, old, gain[:, :1].expand(8, 100), mask=mask[:1].expand(8, 100), ref_logps=ref[:1].expand(8, 100))
    two = TR.policy_loss(logps, old, gain[:, 0], mask=mask[:1].expand(8, 100).contiguous())
    assert torch.equal(one.loss, two.loss) and torch.equal(one.clipped, two.clipped) and two.kl == 0
    x = logps.clone().requires_grad_()

    def call():
        p = TR.policy_loss(x, old, gain, mask=mask, ref_logps=ref, kl_weight=0.1, reduction="sequences")
        q = TR.preference_loss(x, ref, mask)
        return p.loss.detach(), q.loss.detach(), torch.autograd.grad(p.loss + q.loss, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, eager))
    mask.logical_not_()
    with torch.no_grad():
        x.add_(0.1)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, call()))
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(TR.policy_loss(x, old, gain).loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(TR.preference_loss(x, ref).loss, x, create_graph=True)


def test_losses_places_past_32_bits():
    rows, length = 70000, 32768
    logps = torch.zeros(rows, length, dtype=torch.bfloat16, device=DEV)
    logps[-1, -3:] = torch.tensor([-0.5, 0.25, -1.0])
    mask = torch.zeros(rows, length, dtype=torch.bool, device=DEV)
    mask[-1, -3:] = True
    logps.requires_grad_()
    r = TR.preference_loss(logps, None, mask, beta=1.0, reduction="sum")
    grad, = torch.autograd.grad(r.loss, logps)
    assert float(r.rejected_rewards[-1]) == -1.25 and float(grad[-1, -1]) == pytest.approx(float(torch.sigmoid(torch.tensor(-1.25))), rel=2.0 ** -8)
    assert int((grad != 0).sum()) == 3
    del grad, r
    r = TR.policy_loss(logps, None, torch.ones(rows, device=DEV), mask=mask)
    grad, = torch.autograd.grad(r.loss, logps)
    assert float(r.loss.detach()) == -1.0 and grad[-1, -3:].tolist() == pytest.approx([-1 / 3] * 3, rel=2.0 ** -8)


# ---- together ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tuned_with_preferences_then_served_beside_a_packed_projection(dtype):
    """Adapters with dropout, the loss of a head for each token, preference pairs and a clipped policy behind it, fused steps; then a bank that
    serves them in one batch beside a projection of packed weights."""
    from oxibonsai_b200.ops import cuda_ops as K
    torch.manual_seed(0)
    d, vocab, pairs, length = 256, 500, 3, 24
    w = (torch.randn(d, d, device=DEV) / 16).to(dtype)
    head = (torch.randn(vocab, d, device=DEV) / 16).to(dtype)
    adapters = [TR.LoraAdapter(d, d, TR.LoraConfig(rank=r, fused=True, dropout=0.1), seed=r).to(DEV, dtype) for r in (4, 8)]
    x = torch.randn(2 * pairs, length, d, device=DEV).to(dtype)
    tokens = torch.randint(0, vocab, (2 * pairs, length), device=DEV)
    tokens[:, :5] = -100
    mask = tokens >= 0
    for k, adapter in enumerate(adapters):
        torch.nn.init.normal_(adapter.B, std=0.05)
        opt = TR.FusedAdamW(list(adapter.parameters()), lr=1e-2)
        logps = lambda: -TR.linear_cross_entropy(adapter(x, x @ w.T), head, tokens, reduction="none")  # noqa: E731
        with torch.no_grad():
            ref = logps()
        before = [p.detach().clone() for p in adapter.parameters()]
        for _ in range(3):
            l = logps()
            loss = TR.preference_loss(l, ref, mask, beta=0.5).loss if k == 0 else TR.policy_loss(l, ref, torch.randn(2 * pairs, device=DEV), mask=mask, ref_logps=ref, kl_weight=0.1).loss
            opt.zero_grad()
            loss.backward()
            assert all(p.grad.isfinite().all() and p.grad.any() for p in adapter.parameters())
            opt.step(max_norm=1.0)
        assert all(not torch.equal(p, q) for p, q in zip(adapter.parameters(), before))
    # served: f32 activations, as the packed projections take and give them
    bank = TR.AdapterBank(d, d, rank=8, count=4, dtype=torch.float32, device=DEV)
    for i, adapter in zip((1, 3), adapters):
        bank.set(i, adapter.eval())
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 3, (d, d), generator=g) - 1
    packed = K.PlanarWeight.from_tensors(*_planar(codes))
    rows = torch.randn(5, d, device=DEV)
    ids = torch.tensor([1, 3, -1, 3, 0], device=DEV)
    base = torch.stack([K.bitgemv(packed, r) for r in rows])
    y = bank(rows, base, ids, out=base.clone())
    plain = packed.to_f32().double()
    for i, e in enumerate(ids.tolist()):
        want = rows[i].double() @ plain.T
        if e in (1, 3):
            a = adapters[e // 2]
            want = want + (rows[i].double() @ a.A.double().T) @ a.B.double().T * a.config.scale
        assert float((y[i].double() - want.detach()).abs().max()) <= 1e-4 * float(want.detach().abs().max())


def _planar(codes):
    """Ternary codes [n, k] in the planar words and scales of the packed kernels (csrc/cuda/common.cuh)."""
    n, k = codes.shape
    sign, mag = (codes < 0).long(), (codes != 0).long()
    s, m = sign.view(n, k // 16, 16), mag.view(n, k // 16, 16)
    word = torch.zeros(n, k // 16, dtype=torch.int64)
    for i in range(8):
        nib = s[:, :, i] << 3 | s[:, :, i + 8] << 2 | m[:, :, i] << 1 | m[:, :, i + 8]
        word |= nib << 4 * i
    word = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)
    return word.to(DEV), torch.full((n, k // 128), 0.05, dtype=torch.float16, device=DEV)


# ---- what the entry points promise at their edges ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rank", [2, 16, 64, 128])
@pytest.mark.parametrize("n, d, out", [(2, 200, 200), (1100, 200, 15360), (1100, 15360, 200)])
def test_update_rank_values_of_21_bits(n, d, out, rank, dtype):
    """Two rank values of 21 bits (sums of 200 products of 64 to 127) that differ by one term: their difference comes out as it is, in both
    passes and in the sums over rows.  All sums are whole numbers below 2^24, exact in float32, and the results below 2^7 in every type."""
    g = torch.Generator().manual_seed(rank)
    m, j, p, q = 200, 77, n // 3, n - 1
    whole = lambda *shape: torch.randint(64, 128, shape, generator=g).to(DEV, dtype)  # noqa: E731
    zeros = lambda *shape: torch.zeros(shape, dtype=dtype, device=DEV)  # noqa: E731
    base = zeros(n, out)

    def pair(t):                       # along the first axis: a row and the same less one at j
        row = whole(m)
        t[0, ..., :m] = row
        t[1, ..., :m] = row
        t[1, ..., j] -= 1

    x, a, b = zeros(n, d), zeros(1, rank, d), zeros(1, out, rank)
    x[:, :m] = whole(n, m)
    pair(a[0])
    b[0, :, 0], b[0, :, 1] = 1, -1
    for with_base in (base, None):
        y, = run_update(x, with_base, None, a, b, 1.0, None, want="")
        assert torch.equal(y, x[:, j:j + 1].expand(n, out))

    dy, a, b = zeros(n, out), zeros(1, rank, d), zeros(1, out, rank)
    dy[:, :m] = whole(n, m)
    pair(b[0].T)
    a[0, 0], a[0, 1] = 1, -1
    _, dx = run_update(x, base, dy, a, b, 1.0, None, want="x")
    assert torch.equal(dx, dy[:, j:j + 1].expand(n, d))

    x, dy, b = zeros(n, d), zeros(n, out), zeros(1, out, rank)
    x[p], x[q] = 1, -1
    two = zeros(2, out)
    pair(two)
    dy[p], dy[q] = two
    b[0, :m, 0] = whole(m)
    _, da = run_update(x, base, dy, a, b, 1.0, None, want="a")
    assert torch.equal(da[0, 0], b[0, j, 0].expand(d)) and not da[0, 1:].any()

    x, dy, a = zeros(n, d), zeros(n, out), zeros(1, rank, d)
    dy[p], dy[q] = 1, -1
    two = zeros(2, d)
    pair(two)
    x[p], x[q] = two
    a[0, 0, :m] = whole(m)
    _, db = run_update(x, base, dy, a, b, 1.0, None, want="b")
    assert torch.equal(db[0, :, 0], a[0, 0, j].expand(out)) and not db[0, :, 1:].any()



def _groups_that_cancel(groups, total, make, seed):
    """[2 groups + 1, 16, ...] of `make` (groups of 16 whole numbers whose sum is a multiple of 256), the same ones negative in another order, and one that
    leaves ``total``."""
    g = torch.Generator().manual_seed(seed)
    first = make(g, groups)
    return torch.cat([first, -first[torch.randperm(groups, generator=g)], total]).flatten(0, 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, groups, cols, adapters", [(2, 8192, 40, 0), (1100, 1000, 15360, 0), (1100, 1000, 15360, 40)])
def test_update_long_products_are_not_cut_off(n, groups, cols, adapters, dtype):
    """Sums of products of up to 2^16 that pass 2^24 on their way and come back to 768.  What matrix instructions add between two additions in float32 stays below
    2^24, and every group of 16 of them is a multiple of 256: such sums are exact in float32 to 2^32, in any order of groups."""
    def make(g, count):
        x, a = torch.randint(0, 256, (count, 16), generator=g), torch.randint(0, 128, (count, 16), generator=g) * 2 + 1
        inverse = torch.tensor([pow(v, -1, 256) for v in a[:, 15].tolist()])
        x[:, 15] = -(x[:, :15] * a[:, :15]).sum(1) * inverse % 256
        return torch.stack([x, a], 2)

    left = torch.zeros(1, 16, 2, dtype=torch.int64)
    left[0, :3] = 16
    both = _groups_that_cancel(groups, left, make, n)
    x, a = both.unbind(1)
    a = a.abs()
    assert int((x * a).sum()) == 768 and int((x * a).cumsum(0).max()) > 2 ** 27
    k, e = len(x), max(1, adapters)
    x, a = x.to(DEV, dtype).expand(n, k).contiguous(), a.to(DEV, dtype).expand(e, 1, k).contiguous()
    b = torch.ones(e, cols, 1, dtype=dtype, device=DEV)
    ids = torch.arange(n, device=DEV) % e if adapters else None
    base = torch.zeros(n, cols, dtype=dtype, device=DEV)
    y, = run_update(x, base, None, a, b, 1.0, ids, want="")
    assert (y == 768).all()
    # the gradient of the rows is the same product: dy as x, b as a
    _, dx = run_update(base, torch.zeros_like(x), x, b.transpose(1, 2).contiguous(), a.transpose(1, 2).contiguous(), 1.0, ids, want="x")
    assert (dx == 768).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rank", [3, 64])
def test_update_sums_over_rows_are_not_cut_off(rank, dtype):
    """As above, over 16 400 rows whose rank values have 17 bits."""
    def make(g, count):
        parts = torch.randint(0, 256, (count, 16, 3), generator=g)
        parts[:, 15, 0] = -parts[:, :15, 0].sum(1) % 256
        return parts

    left = torch.zeros(1, 16, 3, dtype=torch.int64)
    left[0, 4, 1] = 3
    rows = _groups_that_cancel(512, left, make, rank).to(DEV, dtype)
    n = len(rows)
    weight = torch.tensor([1, 256, 256], device=DEV, dtype=dtype)
    assert float((rows.double() @ weight.double()).sum()) == 768 and float((rows.double() @ weight.double()).cumsum(0).max()) > 2 ** 28
    ones = torch.ones(n, 40, dtype=dtype, device=DEV)
    b = torch.zeros(1, 3, rank, dtype=dtype, device=DEV)
    b[0, :, 1] = weight
    _, da = run_update(ones, None, rows, torch.zeros(1, rank, 40, dtype=dtype, device=DEV), b, 1.0, None, want="a")
    assert (da[0, 1] == 768).all() and not da[0, 2:].any()
    _, db = run_update(rows, None, ones, b.transpose(1, 2).contiguous(), torch.zeros(1, 40, rank, dtype=dtype, device=DEV), 1.0, None, want="b")
    assert (db[0, :, 1] == 768).all() and not db[0, :, 2:].any()


def test_hinge_at_its_corner():
    for kind, margin, slope in ((torch.float32, 1.0, 0.0), (torch.bfloat16, 1.0, 0.0), (torch.float32, 1.0 - 2.0 ** -24, -0.5)):
        x = torch.tensor([[2 * margin], [0.0]], device=DEV).to(kind).requires_grad_()
        r = TR.preference_loss(x, None, beta=0.5, kind="hinge")
        assert float(r.loss.detach()) == 1.0 - margin and torch.autograd.grad(r.loss, x)[0].flatten().tolist() == [slope, -slope]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, out", [(5, 64), (5, 33), (300, 40), (1100, 15360), (1100, 15361)])
def test_update_leaves_the_sign_of_zeros_in_rows_without_an_adapter(n, out, dtype):
    x, base, _, a, b, scales, ids = update_inputs(n, 16, out, 4, 3, dtype, DEV, seed=n, bare=0.4)
    ids[::2] = -1                                  # tiles of such rows alone, and rows beside others
    base[:, ::2] = -0.0
    y = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales)
    kind = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(y[ids < 0].view(kind), base[ids < 0].view(kind))


@pytest.mark.parametrize("dtype", TYPES)
def test_preference_differences_are_not_rounded(dtype):
    """l - ref of -1 + 2^-30 a thousand times, and 1024: what is left, 2^-20, is lost where each difference is rounded to float32."""
    logps, ref = torch.full((2, 1025), -1.0, device=DEV).to(dtype), torch.full((2, 1025), -2.0 ** -20 if dtype == torch.float16 else -2.0 ** -30, device=DEV).to(dtype)
    logps[:, 0], ref[:, 0] = 1024, 0
    logps[1], ref[1] = 0, 0
    r = TR.preference_loss(logps, ref, beta=1.0)
    step = 2.0 ** -10 if dtype == torch.float16 else 2.0 ** -20
    assert float(r.chosen_rewards[0]) == step


def test_forward_mode_is_refused():
    """A dual tensor needs no requires_grad: the kernels, which would drop its tangent, refuse it wherever it comes in."""
    import torch.autograd.forward_ad as fw
    x, base, dy, a, b, scales, ids = update_inputs(4, 16, 8, 2, 3, torch.float32, DEV)
    logps, old, ref, mask, gain = loss_inputs(4, 6, torch.float32, DEV)
    update = dict(x=x, a=a, b=b, base=base, ids=ids, scale=scales)
    policy = dict(logps=logps, old_logps=old, advantages=gain, mask=mask, ref_logps=ref, kl_weight=0.1)
    bank = TR.AdapterBank(16, 8, rank=2, count=3, dtype=torch.float32, device=DEV)
    v, w = x.clone().requires_grad_(), logps.clone().requires_grad_()
    y, z, loss = TR.dropout(v, 0.5, seed=1), TR.low_rank_update(**{**update, "x": v}), TR.preference_loss(w, ref, mask).loss
    want = TR.low_rank_update(**update), TR.policy_loss(**policy).loss, TR.dropout(x, 0.5, seed=1)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in [lambda: TR.dropout(dual(x), 0.5, seed=1), lambda: TR.preference_loss(dual(logps), ref, mask), lambda: bank(dual(x), base, ids),
                     *(lambda k=k: TR.low_rank_update(**{**update, k: dual(update[k])}) for k in ("x", "a", "b", "base")),
                     lambda: TR.policy_loss(**{**policy, "logps": dual(logps)})]:
            with pytest.raises(NotImplementedError):
                call()
        for call in [lambda: TR.low_rank_update(**{**update, "scale": dual(scales)}), lambda: TR.preference_loss(logps, dual(ref), mask),
                     lambda: TR.low_rank_update(**update, out=dual(torch.empty_like(base))), lambda: TR.low_rank_update(**{**update, "x": dual(x)}, out=torch.empty_like(base)),
                     *(lambda k=k: TR.policy_loss(**{**policy, k: dual(policy[k])}) for k in ("old_logps", "advantages", "ref_logps"))]:
            with pytest.raises(ValueError):
                call()
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, v, dual(x))
        for out, leaf, up in ((z, v, dy), (loss, w, torch.ones_like(loss))):
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad(out, leaf, dual(up))
        got = TR.low_rank_update(**update), TR.policy_loss(**policy).loss, TR.dropout(x, 0.5, seed=1)          # others pass
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_update_out_with_a_history_is_refused_on_the_gpu():
    x, base, _, a, b, scales, ids = update_inputs(5, 12, 7, 4, 2, torch.float32, DEV)
    w = torch.ones(5, 7, device=DEV, requires_grad=True)
    for out in (w, w * 2, w[:], (w * 2).T.contiguous().T[:, :]):
        with pytest.raises(ValueError):
            TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, out=out)
    assert torch.equal(w.detach(), torch.ones_like(w))
    want = TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales)
    with torch.no_grad():
        assert torch.equal(TR.low_rank_update(x, a, b, base=base, ids=ids, scale=scales, out=w), want)


@pytest.mark.parametrize("fused", [True, False])
def test_adapter_with_a_seed_in_a_graph(fused):
    adapter = TR.LoraAdapter(64, 48, TR.LoraConfig(rank=4, fused=fused, dropout=0.5)).to(DEV)
    torch.nn.init.normal_(adapter.B)
    x, base, seed = torch.randn(33, 64, device=DEV), torch.zeros(33, 48, device=DEV), torch.tensor(1, device=DEV)

    def call(v):
        y = adapter(v, base, seed=seed)
        return y.detach(), torch.autograd.grad(y.sum(), v)[0]

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        call(x.clone().requires_grad_())
    torch.cuda.current_stream().wait_stream(warm)
    v = x.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(v)
    seen = []
    for k in (1, 9):
        seed.fill_(k)
        graph.replay()
        seen.append(held[0].clone())
        want = call(x.clone().requires_grad_())
        assert all(torch.equal(p, q) for p, q in zip(held, want))
    assert not torch.equal(*seen)


@pytest.mark.parametrize("fused", [True, False])
def test_adapter_in_a_segment_that_runs_again_on_the_gpu(fused):
    """The update is linear in x: the product of x and its gradient is the sum of the results, with the same mask in both passes alone."""
    adapter = TR.LoraAdapter(64, 48, TR.LoraConfig(rank=4, fused=fused, dropout=0.5)).to(DEV)
    torch.nn.init.normal_(adapter.B)
    x, base = torch.rand(33, 64, device=DEV) + 0.5, torch.zeros(33, 48, device=DEV)
    for seed in (None, 5, torch.tensor(6, device=DEV)):
        v = x.clone().requires_grad_()
        y = TR.checkpoint(lambda t: adapter(t, base, seed=seed), v)
        drawn = torch.cuda.get_rng_state(), torch.get_rng_state()
        grad, = torch.autograd.grad(y.sum(), v)
        assert all(torch.equal(p, q) for p, q in zip(drawn, (torch.cuda.get_rng_state(), torch.get_rng_state())))
        size = float(((x @ adapter.A.T).abs() @ adapter.B.abs().T).sum().detach())
        assert abs(float(y.detach().sum() - (grad * x).sum())) <= 2.0 ** -16 * size           # 2^12 sums of 64 values in float32


def test_a_segment_that_runs_again_in_a_graph():
    """Captured: a fused adapter draws its seed from the CPU's generator, which both runs see alike; one with a seed in a tensor follows the tensor."""
    adapter = TR.LoraAdapter(64, 48, TR.LoraConfig(rank=4, fused=True, dropout=0.5)).to(DEV)
    torch.nn.init.normal_(adapter.B)
    x, base, seed = torch.rand(33, 64, device=DEV) + 0.5, torch.zeros(33, 48, device=DEV), torch.tensor(1, device=DEV)

    def call(v, s):
        y = TR.checkpoint(lambda t: adapter(t, base, seed=s), v)
        return y.detach(), torch.autograd.grad(y.sum(), v)[0]

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        call(x.clone().requires_grad_(), None)
    torch.cuda.current_stream().wait_stream(warm)
    size = float(((x @ adapter.A.T).abs() @ adapter.B.abs().T).sum().detach())
    for s in (None, seed):
        v = x.clone().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, grad = call(v, s)
        seen = []
        for k in (1, 9):
            seed.fill_(k)
            graph.replay()
            assert abs(float(y.sum() - (grad * x).sum())) <= 2.0 ** -16 * size
            seen.append(y.clone())
        assert torch.equal(*seen) == (s is None)
