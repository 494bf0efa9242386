"""Host side of the streaming operators where a call is refused or its inputs
change between calls: what a failing call leaves behind, and what arguments
may be.  No GPU: host-side pools, stand-ins for the launches, or tensors that
have a device but no memory."""
import pytest
import torch

import fastest_flash_attention_b200 as ffa


def _cache(pages=8, ps=4):
    return ffa.PagedKVCache(max_pages=pages, page_size=ps, num_heads=2, head_dim=4, dtype=torch.float32)


def _tokens(n, base=0):
    k = (torch.arange(n, dtype=torch.float32) + base)[None, :, None].expand(2, n, 4).contiguous()
    return k, -k


def test_append_without_enough_pages_changes_nothing():
    c = _cache(pages=3)
    with pytest.raises(RuntimeError, match="out of physical pages"):
        c.append_tokens(0, *_tokens(13))
    assert not c.sequences and c.free_pages == [0, 1, 2]
    c.append_tokens(0, *_tokens(5))
    with pytest.raises(RuntimeError, match="out of physical pages"):
        c.append_tokens(0, *_tokens(8, 5))
    assert c.sequences[0]["len"] == 5 and c.sequences[0]["page_table"] == [0, 1] and c.free_pages == [2]
    c.append_tokens(0, *_tokens(7, 5))  # what fits still does
    assert c.get_kv(0)[0][0, :, 0].tolist() == list(range(12))


class _HostAttention(ffa.FastestFlashStreamingGQA):
    """The module with plain projections for its two launches, so its decoder's bookkeeping runs on the host."""

    def qkv(self, x, start=0):
        B, S, _ = x.shape
        return tuple(p(x).view(B, S, -1, self.head_dim).transpose(1, 2) for p in (self.q_proj, self.k_proj, self.v_proj))

    def attend(self, q, k, v):
        B, H, S, D = q.shape
        return self.o_proj(q.transpose(1, 2).reshape(B, S, H * D))


def _decoder(pages=8, ps=4, window=6, sinks=2, max_len=64):
    torch.manual_seed(0)
    m = _HostAttention(16, 2, 1, 8, sliding_window=window, sink_tokens=sinks, max_len=max_len).eval()
    return ffa.StreamingDecoder(m, max_pages=pages, page_size=ps)


def _unchanged(dec, call, err, match=None):
    """`call` raises and leaves the decoder's cache as it was."""
    c = dec.cache
    before = ({s: dict(q, page_table=list(q["page_table"])) for s, q in c.sequences.items()}, list(c.free_pages),
              dict(c._more_owners), c.k_pages.clone())
    with pytest.raises(err, match=match):
        call()
    assert (c.sequences, c.free_pages, c._more_owners) == before[:3] and torch.equal(c.k_pages, before[3])


@pytest.mark.parametrize("ids", [[0], [0, 1, 2], [3, 3], []])
def test_prefill_takes_one_new_sequence_per_prompt(ids):
    dec = _decoder()
    _unchanged(dec, lambda: dec.prefill(torch.randn(2, 5, 16), ids), ValueError)
    dec.prefill(torch.randn(2, 5, 16), [0, 1])
    assert dec.cache.position(0) == dec.cache.position(1) == 5


@pytest.mark.parametrize("rows,ids", [(1, [0, 1]), (2, [0]), (2, [1, 1]), (0, [])])
def test_step_takes_one_sequence_per_row(rows, ids):
    dec = _decoder()
    dec.prefill(torch.randn(2, 5, 16), [0, 1])
    _unchanged(dec, lambda: dec.step(torch.randn(rows, 1, 16), ids), ValueError, "sequence")


def test_step_takes_one_token_per_row():
    dec = _decoder()
    dec.prefill(torch.randn(2, 5, 16), [0, 1])
    _unchanged(dec, lambda: dec.step(torch.randn(2, 2, 16), [0, 1]), ValueError)


@pytest.mark.parametrize("prompt", [3, 4, 5])
def test_step_that_fails_changes_nothing(prompt):
    """A launch that refuses (here: for tensors without a GPU) comes after the slots were assigned."""
    dec = _decoder()
    dec.prefill(torch.randn(2, prompt, 16), [0, 1])
    _unchanged(dec, lambda: dec.step(torch.randn(3, 1, 16), [0, 5, 1]), RuntimeError, "CUDA")
    _unchanged(dec, lambda: dec.step(torch.randn(2, 1, 16, dtype=torch.float64), [0, 1]), RuntimeError, "dtype")


def test_prefill_that_fails_changes_nothing():
    dec = _decoder(pages=8, ps=4)
    dec.prefill(torch.randn(1, 10, 16), [9])  # 3 pages
    _unchanged(dec, lambda: dec.prefill(torch.randn(3, 8, 16), [0, 1, 2]), RuntimeError, "out of physical pages")
    _unchanged(dec, lambda: dec.prefill(torch.randn(1, 65, 16), [0]), ValueError)  # past the rotary tables
    dec.attn.attend = lambda q, k, v: (_ for _ in ()).throw(RuntimeError("refused"))
    _unchanged(dec, lambda: dec.prefill(torch.randn(1, 8, 16), [0]), RuntimeError, "refused")
    del dec.attn.attend
    dec.prefill(torch.randn(2, 8, 16), [0, 1])
    assert dec.cache.num_free_pages == 8 - 3 - 4


@pytest.mark.parametrize("ps,window,sinks,n", [(4, 6, 2, 30), (4, 6, 0, 30), (4, 1, 9, 40), (4, 100, 2, 30), (4, 3, 50, 20),
                                               (1, 3, 2, 9), (16, 5, 3, 15), (4, 6, 2, 1)])
def test_prefill_leaves_what_append_and_trim_leave(ps, window, sinks, n):
    x = torch.randn(1, n, 16)
    a, b = _decoder(64, ps, window, sinks), _decoder(64, ps, window, sinks)
    out = a.prefill(x, [0])
    q, k, v = b.attn.qkv(x)
    b.cache.append_tokens(0, k[0], v[0])
    b.cache.trim_sequence(0, window, sinks)
    ta, tb = a.cache.sequences[0]["page_table"], b.cache.sequences[0]["page_table"]
    assert [p < 0 for p in ta] == [p < 0 for p in tb] and a.cache.position(0) == n == b.cache.position(0)
    for pa, pb in zip(ta, tb):
        if pa >= 0:
            assert torch.equal(a.cache.k_pages[pa], b.cache.k_pages[pb])
            assert torch.equal(a.cache.v_pages[pa], b.cache.v_pages[pb])
    assert torch.equal(out, b.attn.attend(q, k, v)) and a.cache.num_free_pages == b.cache.num_free_pages


def test_prefill_needs_pages_for_the_visible_tokens_alone():
    dec = _decoder(pages=6, ps=4, window=6, sinks=2)
    dec.prefill(torch.randn(2, 40, 16), [0, 1])  # each: the first page and the last two of ten
    assert dec.cache.num_free_pages == 0
    dec.cache.free_sequence(0)
    dec.cache.free_sequence(1)
    assert sorted(dec.cache.free_pages) == list(range(6))


def _captured_step(monkeypatch, dec, x, ids):
    """The q, k, v that a step projects (its launches replaced on the host)."""
    from fastest_flash_attention_b200 import streaming
    seen = {}

    def append(q, k, v, *args, **kw):
        seen.update(q=q, k=k, v=v)
        return q
    monkeypatch.setattr(streaming, "rotary_append", append)
    monkeypatch.setattr(streaming, "paged_decode", lambda q, *args, **kw: q)
    dec.step(x, ids)
    return seen


@pytest.mark.parametrize("bias", [False, True])
def test_step_uses_the_weights_of_its_own_time(monkeypatch, bias):
    """Weights written through .data change neither address nor version."""
    dec = _decoder()
    m = dec.attn
    if bias:
        for p in (m.q_proj, m.k_proj, m.v_proj):
            p.bias = torch.nn.Parameter(torch.randn(p.out_features))
    dec.prefill(torch.randn(2, 5, 16), [0, 1])
    for change in (lambda t: None, lambda t: t.data.mul_(-2.0), lambda t: t.data.copy_(torch.randn_like(t))):
        for p in (m.q_proj, m.k_proj, m.v_proj):
            for t in p.parameters():
                change(t)
        x = torch.randn(2, 1, 16)
        got = _captured_step(monkeypatch, dec, x, [0, 1])
        for name, n in (("q", 2), ("k", 1), ("v", 1)):
            want = getattr(m, name + "_proj")(x[:, 0]).view(2, n, 8)
            # 16 products of fp32 values, summed in another order at most
            torch.testing.assert_close(got[name], want, rtol=1e-5, atol=1e-5)


def test_step_with_parameters_made_in_inference_mode(monkeypatch):
    with torch.inference_mode():
        dec = _decoder()
        dec.prefill(torch.randn(1, 5, 16), [0])
        assert _captured_step(monkeypatch, dec, torch.randn(1, 1, 16), [0])["q"].shape == (1, 2, 8)


def test_tables_built_in_inference_mode_serve_training_too():
    m = _decoder().attn
    with torch.inference_mode():
        first = m.tables(torch.device("cpu"))
    assert not any(t.is_inference() for t in m.tables(torch.device("cpu")))
    assert all(a is b for a, b in zip(first, m.tables(torch.device("cpu"))))


@pytest.mark.parametrize("k,v", [((2, 5, 4), (2, 3, 4)), ((2, 3, 4), (2, 5, 4)), ((3, 5, 4), (3, 5, 4)),
                                 ((2, 5, 3), (2, 5, 3)), ((2, 5, 4), (2, 5, 8))])
def test_append_of_mismatched_shapes_changes_nothing(k, v):
    """The kernel reads both by one shape: a shorter one would be read past its end."""
    c = _cache()
    c.append_tokens(0, *_tokens(3))
    before = list(c.free_pages), c.k_pages.clone()
    with pytest.raises(ValueError, match="append"):
        c.append_tokens(0, torch.zeros(k), torch.zeros(v))
    with pytest.raises(ValueError, match="append"):
        c.append_tokens(1, torch.zeros(k), torch.zeros(v))
    assert list(c.sequences) == [0] and c.sequences[0]["len"] == 3
    assert c.free_pages == before[0] and torch.equal(c.k_pages, before[1])
    c.append_tokens(0, torch.full((1, 2, 4), 7.0), torch.full((2, 1, 4), 8.0))  # repeated over heads, over tokens
    assert bool((c.get_kv(0)[0][:, 3:] == 7).all()) and bool((c.get_kv(0)[1][:, 3:] == 8).all())


def test_append_whose_write_fails_changes_nothing(monkeypatch):
    c = _cache()
    c.append_tokens(0, *_tokens(3))

    def fail(*args):
        raise RuntimeError("refused")
    monkeypatch.setattr(c, "_write", fail)
    for s in (0, 1):
        with pytest.raises(RuntimeError, match="refused"):
            c.append_tokens(s, *_tokens(9))
        assert list(c.sequences) == [0] and c.sequences[0] == {"page_table": [0], "len": 3}
        assert c.free_pages == list(range(1, 8))


@pytest.mark.parametrize("call", ["fork", "compact"])
def test_fork_or_compaction_whose_copy_fails_changes_nothing(call):
    c = _cache(pages=16)
    c.append_tokens(0, *_tokens(30))
    c.append_tokens(1, *_tokens(6))
    before = {s: dict(q, page_table=list(q["page_table"])) for s, q in c.sequences.items()}
    kept, free, v_pages = c.k_pages[:10].clone(), list(c.free_pages), c.v_pages
    c.v_pages = torch.zeros(1)  # the copy of the values fails
    with pytest.raises((IndexError, RuntimeError)):
        c.fork_sequences([(0, 5), (1, 6)]) if call == "fork" else c.compact_sequences([0, 1], 3, 2)
    c.v_pages = v_pages
    assert c.sequences == before and c.free_pages == free and not c._more_owners
    assert torch.equal(c.k_pages[:10], kept)
    if call == "fork":
        c.fork_sequences([(0, 5), (1, 6)])
        assert c.get_kv(5)[0][0, :, 0].tolist() == list(range(30)) and c.get_kv(6)[1][0, :, 0].tolist()[1:] == [-1, -2, -3, -4, -5]
    else:
        assert c.compact_sequences([0, 1], 3, 2) == 26
        assert c.get_kv(0)[0][0, :, 0].tolist() == [0, 1, 27, 28, 29] and c.get_kv(1)[0][0, :, 0].tolist() == [0, 1, 3, 4, 5]
