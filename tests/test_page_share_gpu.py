"""DevicePageTable.share: rows that begin with another's pages.  What the owner does not
hold, or would be lost, is refused on the device and changes nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _mask(rows, n):
    return torch.tensor([r in rows for r in range(n)], device="cuda")


def _copy(t):
    return [x.clone() for x in (t.block_table, t.ctx_lens, t.free_pages, t.free_state)]


def _table(lens, width=8, pages=64):
    from fastest_flash_attention_b200 import DevicePageTable
    t = DevicePageTable(len(lens), width, pages, page_size=16)
    t.assign(_ints(lens), sum(lens))
    return t


def _refused(t, *args):
    kept = _copy(t)
    with pytest.raises(RuntimeError, match="share"):
        t.share(*args)
    assert all(torch.equal(a, b) for a, b in zip(_copy(t), kept))


def test_owner_that_does_not_hold_the_tokens():
    t = _table([40, 0, 0, 31, 0])
    _refused(t, 3, [1], 32)            # 31 tokens: the second page is not full
    _refused(t, 0, [1, 2], 48)         # a page of 40 tokens in part
    _refused(t, 4, [1], 16)            # nothing was ever there
    t.release(_mask([0], 5))           # a released row keeps its entries, whose pages are free
    assert int(t.block_table[0].max()) >= 0
    _refused(t, 0, [1, 2], 32)
    t.assign(_ints([20, 0, 0, 0, 0]), 20)
    _refused(t, 0, [1, 2], 32)         # now another request's, and shorter
    t.share(0, [1, 2], 16)
    assert t.ctx_lens.tolist() == [20, 16, 16, 31, 0]
    assert bool((t.block_table[1:3, 0] == t.block_table[0, 0]).all())


def test_rows_that_are_not_empty():
    t = _table([64, 0, 5, 0])
    _refused(t, 0, [1, 2, 3], 32)
    _refused(t, 0, [2], 32)
    t.share(0, [1], 32)
    _refused(t, 0, [1, 3], 32)         # shared already: its length stands
    t.release(_mask([1, 2], 4), keep=_ints([0, 32, 0, 0]))
    t.share(0, [2, 1], 64)
    assert t.ctx_lens.tolist() == [64, 64, 64, 0] and t.num_free_pages == 60


def test_entries_outside_the_pool():
    t = _table([64, 0])
    t.block_table[0, 1] = 64
    _refused(t, 0, [1], 32)
    t.block_table[0, 1] = -1
    _refused(t, 0, [1], 32)
    t.share(0, [1], 16)                # (that page is not among these)


def test_an_error_is_recorded_without_the_check(monkeypatch):
    from fastest_flash_attention_b200 import _lib
    t = _table([40, 0, 7])
    kept = _copy(t)
    monkeypatch.setenv("FFA_SYNC_CHECK", "0")
    t.share(1, [0], 16)
    t.share(0, [2], 16)
    with pytest.raises(RuntimeError, match="share"):
        _lib.check_device_errors(t.ctx_lens.device)
    assert all(torch.equal(a, b) for a, b in zip(_copy(t), kept))


@pytest.mark.parametrize("R,width,tokens,owner,rows", [
    (1, 4, 16, 0, []),
    (2, 1, 16, 1, [0]),
    (9, 300, 16 * 257, 4, [8, 0, 3]),              # a piece and one entry more
    (257, 520, 16 * 512, 256, list(range(256))),   # samples of a long prompt
    (16384, 3, 32, 16383, list(range(0, 16383, 3))),
])
def test_against_plain(R, width, tokens, owner, rows):
    from fastest_flash_attention_b200 import DevicePageTable
    t = DevicePageTable(R, width, width + 5, page_size=16)
    new = torch.zeros(R, dtype=torch.int32, device="cuda")
    new[owner] = min(tokens + 7, width * 16)
    t.free_state[0] = 3                            # (the ring wraps)
    t.assign(new, int(new[owner]))
    table, lens = t.block_table.clone(), t.ctx_lens.clone()
    table[rows, :tokens // 16] = table[owner, :tokens // 16].clone()
    lens[rows] = tokens
    t.share(owner, rows, tokens)
    assert torch.equal(t.block_table, table) and torch.equal(t.ctx_lens, lens)


def test_captured_on_a_side_stream():
    """A prompt in, its samples, all out again: every replay does the same as the first."""
    t, w = (_table([0, 0, 0, 0]) for _ in range(2))
    new, done, keep = _ints([0, 50, 0, 0]), _mask(range(4), 4), _ints([48, 0, 48, 0])

    def step(x):
        x.assign(new, 50)
        x.share(1, [2, 0], 48)
        lens = x.ctx_lens.clone()
        same = (x.block_table[:3, :3] == x.block_table[1, :3]).all()
        x.release(done, keep=keep)
        return lens, same
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(w)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        lens, same = step(t)
    for _ in range(40):                            # the ring goes round twice
        g.replay()
        torch.cuda.synchronize()
        assert lens.tolist() == [48, 50, 48, 0] and bool(same)
        assert t.num_free_pages == 64 and t.ctx_lens.tolist() == [0] * 4
    from fastest_flash_attention_b200 import _lib
    _lib.check_device_errors(t.ctx_lens.device)
