"""Page tables built on the device against a plain list-and-deque allocator, and
against the host cache's own order.  All values are whole numbers and equal."""
import random
from collections import deque

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _state(lens, width, ps, P, head, rng, first_free=None):
    """Random tables for lens (-1 behind a row's pages), and the ring of the pages left."""
    ids = list(range(P))
    rng.shuffle(ids)
    table = [[-1] * width for _ in lens]
    for r, n in enumerate(lens):
        for i in range(-(-n // ps)):
            table[r][i] = ids.pop()
    free = deque(ids)
    ring = [-7] * P
    for i, x in enumerate(free):
        ring[(head + i) % P] = x
    return table, free, ring


def _plain_assign(table, lens, new, free, ps):
    slots, pos, starts = [], [], [0]
    lens = list(lens)
    for r, n in enumerate(new):
        for _ in range(n):
            if lens[r] % ps == 0:
                table[r][lens[r] // ps] = free.popleft()
            slots.append(table[r][lens[r] // ps] * ps + lens[r] % ps)
            pos.append(lens[r])
            lens[r] += 1
        starts.append(len(slots))
    return slots, pos, starts, lens


@pytest.mark.parametrize("lens,new,ps,extra,head", [
    ([0], [1], 16, 0, 0),                                       # one token of one request
    ([5], [0], 16, 3, 2),                                       # nothing to do
    ([0, 16, 15, 17, 0, 31], [1, 1, 1, 15, 0, 1], 16, 9, 40),   # page edges; the ring wraps
    ([3, 0, 900], [5000, 1, 1], 24, 2, 7),                      # a long prompt, page 24
    ([7] * 513, [1] * 513, 8, 0, 600),                          # a row more than a block's threads
    ([1, 0, 2], [3, 4, 0], 1, 5, 0),                            # a page for every token
    ([100] * 3, [70000, 0, 1], 128, 1, 3),
])
@pytest.mark.parametrize("advance", [False, True])
def test_assign(lens, new, ps, extra, head, advance):
    from fastest_flash_attention_b200 import assign_slots
    rng = random.Random(len(lens) + ps)
    width = max(-(-(a + b) // ps) for a, b in zip(lens, new)) + 1
    P = sum(-(-(a + b) // ps) for a, b in zip(lens, new)) + extra
    head %= P
    table, free, ring = _state(lens, width, ps, P, head, rng)
    bt, ln, rg, st = _ints(table), _ints(lens), _ints(ring), _ints([head, len(free)])
    total = sum(new)
    before = len(free)
    slots, pos, starts, after = _plain_assign(table, lens, new, free, ps)
    for tail in (0, 5):
        b, l, s = bt.clone(), ln.clone(), st.clone()
        plan = assign_slots(b, l, _ints(new), rg, s, page_size=ps, max_tokens=total + tail, advance=advance)
        assert plan.slots.tolist() == slots + [-1] * tail and plan.positions.tolist() == pos + [0] * tail
        assert plan.starts.tolist() == starts and plan.ctx_lens.tolist() == after
        assert plan.free_state.tolist() == [(head + before - len(free)) % P, len(free)]
        assert b.tolist() == table and rg.tolist() == ring  # other entries, and the ring, as they were
        if advance:
            assert plan.ctx_lens is l and plan.free_state is s
        else:
            assert torch.equal(l, ln) and torch.equal(s, st)


@pytest.mark.parametrize("R", [1, 4000, 16384])
def test_assign_and_release_many(R):
    from fastest_flash_attention_b200 import assign_slots, release_pages
    rng = random.Random(R)
    ps, width = 16, 12
    lens = [rng.choice([0, 1, 15, 16, 17, rng.randrange(120)]) for _ in range(R)]
    new = [rng.choice([0, 1, 1, rng.randrange(60)]) for _ in range(R)]
    P = R * width + 3
    head = rng.randrange(P)
    table, free, ring = _state(lens, width, ps, P, head, rng)
    bt, rg = _ints(table), _ints(ring)
    slots, pos, starts, after = _plain_assign(table, lens, new, free, ps)
    plan = assign_slots(bt, _ints(lens), torch.tensor(new, device="cuda"), rg, _ints([head, P - sum(-(-n // ps) for n in lens)]),
                        page_size=ps, max_tokens=sum(new))
    assert plan.slots.tolist() == slots and plan.positions.tolist() == pos and plan.starts.tolist() == starts
    assert bt.tolist() == table and plan.ctx_lens.tolist() == after
    done = [rng.random() < 0.6 for _ in range(R)]
    keep = [rng.choice([0, 0, 16, 32, 500]) for _ in range(R)]
    h, c = plan.free_state.tolist()
    for kp in (None, keep):
        r2 = rg.clone()
        lens2, state2 = release_pages(bt, plan.ctx_lens, torch.tensor(done, device="cuda"), r2, plan.free_state,
                                      page_size=ps, keep=None if kp is None else _ints(kp))
        given = [table[r][i] for r in range(R) if done[r]
                 for i in range(-(-(kp[r] if kp else 0) // ps), -(-after[r] // ps))]
        want = rg.tolist()
        for i, x in enumerate(given):
            want[(h + c + i) % P] = x
        assert r2.tolist() == want and state2.tolist() == [h, c + len(given)]
        assert lens2.tolist() == [0 if d else n for d, n in zip(done, after)]
        assert bt.tolist() == table


def test_assign_that_cannot_be_done_changes_nothing():
    from fastest_flash_attention_b200 import assign_slots
    table, free, ring = _state([5, 16], 4, 16, 8, 3, random.Random(0))
    good = dict(lens=[5, 16], new=[20, 1], table=table, ring=ring, state=[3, 6], tokens=21)
    bad_first = [row[:] for row in table]
    bad_first[0][0] = 8  # the page that request 0 goes on in
    for change in (dict(state=[3, 1]), dict(state=[8, 6]), dict(state=[-1, 6]), dict(state=[3, 9]), dict(state=[3, -1]),
                   dict(tokens=20), dict(tokens=0), dict(lens=[-1, 16]), dict(lens=[5, 65]), dict(new=[60, 1]),
                   dict(new=[-1, 1]), dict(new=[2 ** 31 - 1, 2 ** 31 - 1]), dict(ring=[-1] * 8), dict(ring=[8] * 8),
                   dict(table=bad_first)):
        a = dict(good, **change)
        bt, ln, rg, st = (_ints(a[x]) for x in ("table", "lens", "ring", "state"))
        kept = [x.clone() for x in (bt, ln, rg, st)]
        with pytest.raises(RuntimeError, match="assign_slots"):
            assign_slots(bt, ln, _ints(a["new"]), rg, st, page_size=16, max_tokens=a["tokens"], advance=True)
        assert all(torch.equal(x, y) for x, y in zip((bt, ln, rg, st), kept))
    bt, ln, rg, st = (_ints(good[x]) for x in ("table", "lens", "ring", "state"))
    assert assign_slots(bt, ln, _ints([20, 1]), rg, st, page_size=16, max_tokens=21).starts.tolist() == [0, 20, 21]


def test_failed_assign_gives_no_slots(monkeypatch):
    """Without the check after each call: slots -1 and starts 0, so that later launches write and attend nothing."""
    from fastest_flash_attention_b200 import _lib, assign_slots
    monkeypatch.setenv("FFA_SYNC_CHECK", "0")
    bt, ln, rg, st = _ints([[-1, -1]]), _ints([0]), _ints([0, 1]), _ints([0, 1])
    plan = assign_slots(bt, ln, _ints([20]), rg, st, page_size=16, max_tokens=20)
    assert plan.slots.tolist() == [-1] * 20 and plan.positions.tolist() == [0] * 20 and plan.starts.tolist() == [0, 0]
    assert plan.ctx_lens.tolist() == [0] and plan.free_state.tolist() == [0, 1] and bt.tolist() == [[-1, -1]]
    with pytest.raises(RuntimeError, match="free pages"):
        _lib.check_device_errors(ln.device)


def test_release_that_cannot_be_done_changes_nothing():
    from fastest_flash_attention_b200 import release_pages
    table, free, ring = _state([5, 33], 4, 16, 8, 3, random.Random(1))
    good = dict(lens=[5, 33], table=table, ring=ring, state=[3, 4], keep=[0, 0])
    bad_table = [row[:] for row in table]
    bad_table[1][2] = -1
    for change in (dict(state=[3, 5]), dict(state=[8, 4]), dict(lens=[5, 65]), dict(lens=[-1, 33]), dict(keep=[0, -1]),
                   dict(table=bad_table)):
        a = dict(good, **change)
        bt, ln, rg, st = (_ints(a[x]) for x in ("table", "lens", "ring", "state"))
        kept = [x.clone() for x in (bt, ln, rg, st)]
        with pytest.raises(RuntimeError, match="release_pages"):
            release_pages(bt, ln, torch.tensor([True, True], device="cuda"), rg, st, page_size=16, keep=_ints(a["keep"]),
                          advance=True)
        assert all(torch.equal(x, y) for x, y in zip((bt, ln, rg, st), kept))


def test_no_rows_and_no_tokens():
    from fastest_flash_attention_b200 import assign_slots, release_pages
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    bt, rg, st = torch.empty(0, 4, dtype=torch.int32, device="cuda"), _ints([2, 0, 1]), _ints([1, 2])
    plan = assign_slots(bt, none, none, rg, st, page_size=16, max_tokens=0)
    assert plan.starts.tolist() == [0] and plan.slots.numel() == 0 and plan.free_state.tolist() == [1, 2]
    lens, state = release_pages(bt, none, none.bool(), rg, st, page_size=16)
    assert lens.numel() == 0 and state.tolist() == [1, 2]


def test_same_order_as_the_host_cache():
    """A run of appends and frees: the same tables as PagedKVCache's, page by page."""
    from fastest_flash_attention_b200 import DevicePageTable, PagedKVCache
    rng = random.Random(5)
    host = PagedKVCache(max_pages=60, page_size=4, num_heads=1, head_dim=8, dtype=torch.float16, device="cuda")
    dev = DevicePageTable(6, 16, 60, page_size=4)
    for _ in range(25):
        new = [rng.choice([0, 0, 1, 3, 9]) for _ in range(6)]
        lens = [host.sequences.get(r, {"len": 0})["len"] for r in range(6)]
        new = [n if a + n <= 64 else 0 for a, n in zip(lens, new)]
        need = sum(-(-(a + n) // 4) + a // -4 for a, n in zip(lens, new))
        if need <= host.num_free_pages:
            slots = [s for r, n in enumerate(new) if n for s in host._assign_slots(r, n)]
            assert dev.assign(_ints(new), 60).slots.tolist()[:len(slots)] == slots
        done = [rng.random() < 0.2 for _ in range(6)]
        for r in range(6):
            if done[r]:
                host.free_sequence(r)
        dev.release(torch.tensor(done, device="cuda"))
        assert dev.num_free_pages == host.num_free_pages
        h, c = dev.free_state.tolist()
        assert [dev.free_pages.tolist()[(h + i) % 60] for i in range(c)] == host.free_pages
        for r in range(6):
            pages = host.sequences.get(r, {"page_table": []})["page_table"]
            assert dev.block_table[r, :len(pages)].tolist() == pages


def test_shared_prefix_and_its_release():
    from fastest_flash_attention_b200 import DevicePageTable
    t = DevicePageTable(4, 8, 20, page_size=16)
    t.assign(_ints([40, 0, 0, 0]), 40)
    t.share(0, [1, 3], 32)
    plan = t.assign(_ints([0, 5, 0, 1]), 6)
    assert t.ctx_lens.tolist() == [40, 37, 0, 33] and plan.positions.tolist() == [32, 33, 34, 35, 36, 32]
    assert t.block_table[1, :3].tolist() == [0, 1, 3] and t.block_table[3, :3].tolist() == [0, 1, 4]
    t.release(torch.tensor([False, True, False, True], device="cuda"), keep=_ints([0, 32, 0, 32]))
    assert t.num_free_pages == 17 and t.ctx_lens.tolist() == [40, 0, 0, 0]
    t.release(torch.tensor([True, False, False, False], device="cuda"))
    assert t.num_free_pages == 20 and sorted(t.free_pages.tolist()) == list(range(20))
    for owner, rows, tokens in ((0, [1], 5), (0, [1], 0), (0, [0], 16), (0, [1, 1], 16), (0, [4], 16), (4, [1], 16),
                                (0, [1], 16 * 9)):
        with pytest.raises(ValueError):
            t.share(owner, rows, tokens)


def test_captured_steps():
    """Assign and release in a graph on a side stream, replayed: every replay goes on from the last."""
    from fastest_flash_attention_b200 import DevicePageTable
    t, w = (DevicePageTable(3, 40, 64, page_size=4) for _ in range(2))
    new, done = _ints([1, 2, 0]), torch.tensor([False, True, False], device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        w.assign(new, 3)
        w.release(done)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        plan = t.assign(new, 3)
        t.release(done)
    for i in range(9):
        g.replay()
        torch.cuda.synchronize()
        assert t.ctx_lens.tolist() == [i + 1, 0, 0] and plan.positions.tolist() == [i, 0, 1]
        assert t.num_free_pages == 64 - (i // 4 + 1)
