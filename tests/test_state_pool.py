"""Slots of pools of states: refusals (CPU); copies and compactions against lists (GPU). Rows are copied bit by bit: everything is
compared for equality."""

import pytest
import torch

from nvsubquadratic_b200.state_pool import compact_slots, copy_slots

gpu = pytest.mark.gpu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32)


def _copied(pool, source, target):
    """The definition, one move after the other from a second buffer."""
    out = pool.clone()
    for s, t in zip(source, target):
        if 0 <= t < len(pool):
            out[t] = pool[s] if 0 <= s < len(pool) else 0
    return out


def test_refusals():
    p, i = torch.zeros(4, 8), _i32([0, 1])
    with pytest.raises(RuntimeError, match="CUDA"):
        copy_slots(p, i, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        compact_slots(p, torch.ones(4, dtype=torch.bool))
    with pytest.raises(AssertionError, match="same slots"):
        copy_slots([p, torch.zeros(5)], i, i)
    with pytest.raises(AssertionError, match="1 to 16 pools"):
        copy_slots([], i, i)
    with pytest.raises(AssertionError, match="1 to 16 pools"):
        copy_slots([p] * 17, i, i)
    with pytest.raises(AssertionError, match="contiguous"):
        copy_slots(p.t(), i, i)
    with pytest.raises(AssertionError, match="source must be int32"):
        copy_slots(p, i.long(), i)
    with pytest.raises(AssertionError, match=r"target must be \[n\]"):
        copy_slots(p, i, i[None])
    with pytest.raises(AssertionError, match="agree"):
        copy_slots(p, i, i[:1])
    with pytest.raises(AssertionError, match="live must be bool"):
        compact_slots(p, torch.ones(4))
    with pytest.raises(AssertionError, match=r"live must be \[4\]"):
        compact_slots(p, torch.ones(3, dtype=torch.bool))
    with pytest.raises(NotImplementedError, match="gradient"):
        copy_slots(p.clone().requires_grad_(), i, i)


def test_library_refuses_what_it_cannot_hold():
    """Checked on the host, before anything is launched."""
    import ctypes

    from nvsubquadratic_b200 import _lib

    lib, one = _lib.load(), (_lib.Pool * 1)(_lib.Pool(16, 16))
    buf = ctypes.c_void_p(16)
    assert lib.hyfft_pool_copy(one, 1, 4, buf, buf, 12801, buf, 1 << 30, None) == _lib.HYFFT_ERR_UNSUPPORTED
    assert lib.hyfft_pool_copy(one, 1, 4, buf, buf, 2, buf, 8, None) == _lib.HYFFT_ERR_WORKSPACE
    assert lib.hyfft_pool_copy(one, 1, 0, buf, buf, 2, buf, 1 << 30, None) == _lib.HYFFT_ERR_INVALID
    assert lib.hyfft_pool_copy(one, 17, 4, buf, buf, 2, buf, 1 << 30, None) == _lib.HYFFT_ERR_INVALID
    assert lib.hyfft_pool_compact(one, 1, 4, None, buf, buf, 1 << 30, None) == _lib.HYFFT_ERR_INVALID
    assert lib.hyfft_pool_copy(one, 1, 4, buf, buf, 0, None, 0, None) == _lib.HYFFT_OK


# rows: of 4, 2, 4 (odd numbers of), 8, 1 and many bytes
def _make(slots, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(slots, 3, 40, generator=g), torch.randint(-9, 9, (slots, 7), generator=g).to(torch.int16),
            torch.randn(slots, 33, generator=g), torch.randint(0, 1 << 40, (slots,), generator=g), torch.rand(slots, 5, generator=g) < 0.5,
            torch.randn(slots, 5000, generator=g).bfloat16()]


CASES = {
    "fork": ([3, 3, 3, 5], [0, 9, 1, 2]),
    "exchange": ([1, 2], [2, 1]),
    "cycle and chain": ([1, 2, 0, 4, 5, 6], [0, 1, 2, 3, 4, 5]),
    "itself": ([4, 5], [4, 6]),
    "clear": ([-1, 12, 3], [0, 1, 2]),
    "no target": ([1, 2, 3], [-1, 10, 4]),
    "the last of several": ([1, 2, 3, 4, -1], [7, 7, 7, 8, 8]),
    "the last stays": ([1, 7], [7, 7]),
    "all": (list(range(9, -1, -1)), list(range(10))),
    "none": ([], []),
}


@gpu
@pytest.mark.parametrize("name", CASES)
def test_copies(name):
    source, target = CASES[name]
    pools = _make(10)
    want = [_copied(p, source, target) for p in pools]
    got = [p.cuda() for p in pools]
    copy_slots(got, _i32(source).cuda(), _i32(target).cuda())
    for w, g in zip(want, got):
        assert torch.equal(w, g.cpu())
    one = pools[0].cuda()
    copy_slots(one, _i32(source).cuda(), _i32(target).cuda())
    assert torch.equal(want[0], one.cpu())


@gpu
@pytest.mark.parametrize("slots,moves,row", [(1, 1, 1), (300, 300, 1000), (5000, 4999, 37), (2000, 12800, 12), (64, 3, 300000),
                                             (3000, 3000, 16)])
def test_many_and_large(slots, moves, row):
    g = torch.Generator().manual_seed(slots)
    pools = [torch.randn(slots, row, generator=g), torch.randint(0, 99, (slots,), generator=g)]
    source = torch.randint(-2, slots + 2, (moves,), generator=g).to(torch.int32)
    target = torch.randint(-2, slots + 2, (moves,), generator=g).to(torch.int32)
    held = torch.arange(slots)
    for s, t in zip(source.tolist(), target.tolist()):
        if 0 <= t < slots:
            held[t] = s if 0 <= s < slots else -1
    got = [p.cuda() for p in pools]
    copy_slots(got, source.cuda(), target.cuda())
    for p, g in zip(pools, got):
        want = p[held.clamp(min=0)]
        want[held < 0] = 0
        assert torch.equal(want, g.cpu())


@gpu
def test_too_many_moves_are_refused():
    p, i = torch.zeros(10, 4, device="cuda"), torch.zeros(12801, dtype=torch.int32, device="cuda")
    with pytest.raises(NotImplementedError, match="12800"):
        copy_slots(p, i, i)


@gpu
def test_views_and_unaligned_pools():
    """Part of a larger pool, a pool off 16 bytes, lists with strides; what lies around is left alone."""
    big, off = torch.randn(12, 24), torch.randn(1 + 10 * 24)
    b, o = big.cuda(), off.cuda()
    source, target = _i32([[3, 0], [1, 0], [0, 0]]).cuda()[:, 0], _i32([0, 3, 9]).cuda()
    copy_slots([b[1:11], o[1:].view(10, 24)], source, target)
    assert torch.equal(b.cpu(), torch.cat((big[:1], _copied(big[1:11], [3, 1, 0], [0, 3, 9]), big[11:])))
    assert torch.equal(o.cpu()[1:].view(10, 24), _copied(off[1:].view(10, 24), [3, 1, 0], [0, 3, 9])) and o[0].item() == off[0].item()


def _compacted(pools, live):
    n, slots = sum(live), len(live)
    movers, new, pools = [i for i in range(n, slots) if live[i]], [i if on else -1 for i, on in enumerate(live)], [p.clone() for p in pools]
    for hole in (i for i in range(n) if not live[i]):
        m = movers.pop(0)
        new[m] = hole
        for p in pools:
            p[hole] = p[m]
    return pools, new


@gpu
@pytest.mark.parametrize("slots", [1, 2, 10, 1023, 1024, 2500])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 0.9, 1.0])
def test_compaction(slots, share):
    pools = [torch.randn(slots, 9), torch.arange(slots), torch.randn(slots, 8).bfloat16()]
    live = torch.rand(slots, generator=torch.Generator().manual_seed(slots)) < share
    if share == 0.5:  # the free ones first
        live = torch.arange(slots) >= slots // 2
    want, new = _compacted(pools, live.tolist())
    got = [p.cuda() for p in pools]
    moved = compact_slots(got, live.cuda())
    assert moved.dtype == torch.int32 and moved.tolist() == new
    for w, g in zip(want, got):
        assert torch.equal(w, g.cpu())


@gpu
def test_compaction_of_long_rows_and_of_nothing():
    pools = _make(10) + [torch.randn(10, 70001)]
    live = torch.tensor([0, 1, 0, 0, 1, 1, 0, 1, 0, 1], dtype=torch.bool)
    want, new = _compacted(pools, live.tolist())
    got = [p.cuda() for p in pools]
    assert compact_slots(got, live.cuda()).tolist() == new
    assert all(torch.equal(w, g.cpu()) for w, g in zip(want, got))
    assert compact_slots(torch.zeros(10, 0, device="cuda"), live.cuda()).tolist() == new
    assert compact_slots(torch.zeros(0, 4, device="cuda"), live[:0].cuda()).shape == (0,)
    copy_slots(torch.zeros(0, 4, device="cuda"), _i32([1]).cuda(), _i32([0]).cuda())
    copy_slots(torch.zeros(4, 0, device="cuda"), _i32([1]).cuda(), _i32([0]).cuda())


@gpu
def test_graphs_and_streams():
    """Captured and replayed with other lists; on a stream of its own."""
    pool = torch.randn(50, 700)
    g, source, target = pool.cuda(), torch.arange(50, dtype=torch.int32, device="cuda"), torch.arange(50, dtype=torch.int32, device="cuda")
    live = torch.ones(50, dtype=torch.bool, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        copy_slots(g, source, target)
        compact_slots(g, live)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(g.cpu(), pool)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_slots(g, source, target)
        moved = compact_slots(g, live)
    source.copy_(torch.randperm(50))
    live[::3] = False
    want, new = _compacted([_copied(pool, source.tolist(), target.tolist())], live.tolist())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(g.cpu(), want[0]) and moved.tolist() == new


def test_what_stands_in_for_rows_of_no_bytes_lives_through_the_call(monkeypatch):
    """On the host, with a library that only looks: every tensor whose address it is given is still there."""
    import weakref

    from nvsubquadratic_b200 import _lib, state_pool

    given, alive = [], []

    class Looks:
        def hyfft_pool_workspace_size(self, slots, moves, copy, compact):
            copy._obj.value, compact._obj.value = 4 * (slots + 2 * moves), 4 * (2 * slots + 1)
            return 0

        def hyfft_pool_compact(self, table, count, *rest):
            assert count == 1
            alive.append(all(t() is not None and t().data_ptr() == table[0].data for t in given))
            return 0

    table = state_pool._table

    def remembered(pools):
        given[:] = [weakref.ref(t) for t in pools if t.numel()]
        return table(pools)

    monkeypatch.setattr(state_pool, "_table", remembered)
    monkeypatch.setattr(_lib, "load", Looks)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "stream_ptr", lambda dev: 0)
    for pool in (torch.zeros(50, 0), torch.zeros(50, 3)):
        compact_slots(pool, torch.ones(50, dtype=torch.bool))
    assert alive == [True, True]


@gpu
def test_compaction_of_many_slots_of_no_bytes():
    g = torch.Generator().manual_seed(0)
    for slots in (1500, 20000, 50000):
        live = torch.rand(slots, generator=g) < 0.5
        want = _compacted([], live.tolist())[1]
        for _ in range(3):
            assert compact_slots(torch.zeros(slots, 0, device="cuda"), live.cuda()).tolist() == want
