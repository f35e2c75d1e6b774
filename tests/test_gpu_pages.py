"""Forking, reserving, copying and freeing pages against loops on the host."""
import numpy as np
import pytest
import torch

import logicaffeine_amd as lgx
import tree_ref as ref_

pytestmark = pytest.mark.gpu


class State:
    """The same bookkeeping on the device and on the host."""

    def __init__(self, ctx, pages, S, maxp):
        self.ctx = ctx
        self.ref, self.table, self.lens = np.zeros(pages, np.int32), np.full((S, maxp), -1, np.int32), np.zeros(S, np.int32)
        self.pool = lgx.PagePool.empty(ctx, pages)
        self.dtable, self.dlens = ctx.to_device(self.table.copy()), ctx.to_device(self.lens.copy())

    def check(self):
        assert np.array_equal(self.pool.ref.cpu().numpy(), self.ref)
        assert np.array_equal(self.dtable.cpu().numpy(), self.table)
        assert np.array_equal(self.dlens.cpu().numpy(), self.lens)
        held = self.table[self.table >= 0]
        assert np.array_equal(np.bincount(held, minlength=len(self.ref)), self.ref)

    def i32(self, x):
        return self.ctx.to_device(np.asarray(x, np.int32))

    def fork(self, src, dst):
        self.ctx.pages_fork(self.pool, self.dtable, self.dlens, self.i32(src), self.i32(dst))
        ref_.fork(self.ref, self.table, self.lens, list(src), list(dst))
        self.check()

    def reserve(self, need):
        copies, n, lacking = self.ctx.pages_reserve(self.pool, self.dtable, self.dlens, self.i32(need))
        want, short = ref_.reserve(self.ref, self.table, self.lens, need)
        assert (int(n), int(lacking)) == (len(want), short)
        assert [tuple(x) for x in copies.cpu().tolist()[:len(want)]] == want
        self.check()
        return copies, n, short

    def free(self, keep):
        self.ctx.pages_free(self.pool, self.dtable, self.i32(keep))
        ref_.free(self.ref, self.table, keep)
        self.check()

    def grow(self, by):
        self.lens += np.asarray(by, np.int32)
        self.dlens.copy_(self.ctx.to_device(self.lens))


@pytest.mark.parametrize("pages,S,maxp", [(3, 1, 2), (64, 5, 7), (300, 40, 17), (9000, 70, 300), (20011, 1024, 40)])
def test_a_life_of_forks_reservations_and_ends(ctx, pages, S, maxp):
    rng = np.random.default_rng(pages)
    s = State(ctx, pages, S, maxp)
    for step in range(12):
        need = rng.integers(-3, 40, S)
        need[rng.random(S) < 0.3] = 0
        _, _, short = s.reserve(need)
        room = 16 * maxp - s.lens
        if not short:
            s.grow(np.minimum(np.maximum(need, 0) * (rng.random(S) < 0.8), room))
        s.free(np.where(rng.random(S) < 0.25, 0, s.lens))
        ended = (s.table < 0).all(1)
        s.grow(np.where(ended, -s.lens, 0))
        free_rows, live = np.flatnonzero(s.lens == 0), np.flatnonzero(s.lens > 0)
        if len(free_rows) and len(live):
            dst = rng.permutation(free_rows)[:max(1, len(free_rows) // 2)]
            s.fork(rng.choice(live, len(dst)), dst)


def test_sequences_that_share_a_page_leave_it_in_order(ctx):
    """Of four that write behind the same 20 tokens, the last keeps the page; with
    another holder none does."""
    s = State(ctx, 40, 6, 4)
    s.reserve([20, 0, 0, 0, 0, 0])
    s.grow([20, 0, 0, 0, 0, 0])
    s.fork([0, 0, 0], [1, 3, 5])
    s.reserve([1, 0, 0, 2, 0, 30])                    # row 1 stays a holder: three copies
    s.free([20, 20, 0, 20, 0, 20])
    s.reserve([0, 13, 0, 0, 0, 0])                    # alone by now: no copy
    assert s.ref.max() == 4                           # the full first page


def test_a_reservation_that_lacks_pages_changes_nothing(ctx):
    s = State(ctx, 5, 3, 10)
    assert s.reserve([16, 40, 30])[2] == 1            # 1 + 3 + 2
    assert s.reserve([16, 40, 16])[2] == 0            # exactly all
    assert s.reserve([0, 0, 17])[2] == 1              # one more page for its 17th token
    s.free([0, 0, 0])


def test_tokens_past_the_table_get_no_page(ctx):
    s = State(ctx, 50, 2, 3)
    s.reserve([1000, 2**31 - 1])
    s.grow([48, 48])
    s.reserve([5, 5])


def test_pairs_that_would_race_are_left_out(ctx):
    s = State(ctx, 50, 6, 3)
    s.reserve([40, 17, 3, 0, 0, 0])
    s.grow([40, 17, 3, 0, 0, 0])
    s.fork([0, 1, 0, 2, 7, 0, -1], [3, 3, 1, 2, 4, 9, 5])   # twice to 3, to a source, to itself, outside
    assert s.lens.tolist() == [40, 17, 3, 40, 0, 0]
    s.fork([1, 1], [3, 4])                            # row 3 gives its pages back


def test_entries_outside_the_pool_count_as_none(ctx):
    s = State(ctx, 10, 2, 4)
    s.reserve([16, 16])
    s.table[0, 1], s.table[1, 2] = 10, 2**31 - 1
    s.dtable.copy_(ctx.to_device(s.table))
    got = ctx.pages_reserve(s.pool, s.dtable, s.dlens, s.i32([40, 0]))
    assert int(got[2]) == 0 and s.dtable.cpu().numpy()[0].tolist() == [0, 2, 3, -1]
    ctx.pages_free(s.pool, s.dtable, s.i32([0, 0]))
    assert not s.pool.ref.any() and (s.dtable == -1).all()


@pytest.mark.parametrize("shapes,dtype", [(((3, 16, 64),), torch.int16), (((2, 16, 128), (2,), (5,)), torch.float32),
                                          (((7,), (16,)), torch.int8)])
def test_copies_go_over_every_plane(ctx, shapes, dtype):
    """Planes of pages of any size, 16 bytes a piece or one, and more planes than a
    launch takes."""
    pages = 33
    planes = [torch.randint(-100, 100, (pages, *s), device=ctx.dev).to(dtype) for s in shapes for _ in range(60)]
    want = [p.clone() for p in planes]
    pairs = torch.tensor([[4, 9], [32, 0], [4, 31], [40, 2], [5, -1], [7, 8]], dtype=torch.int32, device=ctx.dev)
    for w in want:
        w[9], w[0], w[31] = w[4], w[32], w[4]         # the sixth is past n_copies
    ctx.pages_copy(lgx.PagePlanes(planes), pairs, torch.tensor([5], dtype=torch.int32, device=ctx.dev))
    for p, w in zip(planes, want):
        assert torch.equal(p, w)
    ctx.pages_copy(lgx.PagePlanes(planes), pairs, torch.zeros(1, dtype=torch.int32, device=ctx.dev))
    for p, w in zip(planes, want):
        assert torch.equal(p, w)


def test_bookkeeping_in_a_graph(ctx):
    """Fork, reserve, copy and free recorded once and replayed, with other work between
    the replays."""
    s = State(ctx, 200, 8, 12)
    s.reserve([100, 50, 16, 7, 0, 0, 0, 0])
    s.grow([100, 50, 16, 7, 0, 0, 0, 0])
    src, dst, need, keep = s.i32([0, 1, 2, 3]), s.i32([4, 5, 6, 7]), s.i32([9] * 8), s.i32([100, 50, 16, 7, 0, 0, 0, 0])
    planes = lgx.PagePlanes([torch.randint(-99, 99, (200, 2, 16, 64), device=ctx.dev, dtype=torch.int16)])
    host = planes.tensors[0].cpu().numpy()
    out = tuple(torch.zeros(n, dtype=torch.int32, device=ctx.dev) for n in ((8, 2), 1, 1))

    def step():
        ctx.pages_fork(s.pool, s.dtable, s.dlens, src, dst)
        ctx.pages_reserve(s.pool, s.dtable, s.dlens, need, out=out)
        ctx.pages_copy(planes, out[0], out[1])
        ctx.pages_free(s.pool, s.dtable, keep)

    def on_host():
        ref_.fork(s.ref, s.table, s.lens, [0, 1, 2, 3], [4, 5, 6, 7])
        copies, lacking = ref_.reserve(s.ref, s.table, s.lens, [9] * 8)
        assert not lacking and copies
        for a, b in copies:
            host[b] = host[a]
        ref_.free(s.ref, s.table, [100, 50, 16, 7, 0, 0, 0, 0])

    step()
    on_host()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        graph.replay()
        on_host()
        torch.cuda.synchronize()
        s.check()
        assert np.array_equal(planes.tensors[0].cpu().numpy(), host)
        ctx.sample_filtered(torch.randn(3, 5000, device=ctx.dev), torch.rand(3, device=ctx.dev))


def test_argument_checks(ctx):
    pool = lgx.PagePool.empty(ctx, 4)
    table = torch.full((2, 3), -1, dtype=torch.int32, device=ctx.dev)
    lens = torch.zeros(2, dtype=torch.int32, device=ctx.dev)
    for bad in (lambda: ctx.pages_reserve(pool, table, lens.long(), lens), lambda: ctx.pages_reserve(pool, table, lens[:1], lens),
                lambda: ctx.pages_reserve(pool, table.t(), lens, lens), lambda: ctx.pages_free(pool, table[0], lens),
                lambda: ctx.pages_fork(pool, table, lens, lens, lens[:1]), lambda: lgx.PagePool(lens.float()),
                lambda: lgx.PagePlanes([]), lambda: lgx.PagePlanes([table, lens[:1]]), lambda: lgx.PagePlanes([table.t()]),
                lambda: ctx.pages_copy(lgx.PagePlanes([table]), lens, lens[:1]),
                lambda: ctx.pages_reserve(pool, table, lens, lens, out=(lens, lens[:1], lens[:1])),
                lambda: ctx.pages_free(pool, table.cpu(), lens)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(AttributeError):
        pool.ref = lens
