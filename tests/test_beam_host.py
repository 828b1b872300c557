"""CPU: refusals and workspace sizes of the shared-prefix attention, beam selection and page re-ordering, which are
decided on the host before any launch; the oracle's own known answers."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import beams

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 4, 5
P = 1 << 20  # an aligned address that no refused call touches


def lib():
    from ssd_b200 import _lib

    return _lib.lib()


def attention(**kw):
    a = dict(stream=None, q=P, pages=P, dtype=0, num_layers=2, num_blocks=64, block_size=16, hkv=2, D=64, layer=1,
             tables=P, max_blocks=8, seq_lens=P, q_lens=None, starts=P, prefixes=P, groups=2, out=P, scale=0.1, B=4, T=2,
             hq=8, max_seq_len=128, ws=P, ws_bytes=0)
    a.update(kw)
    return lib().ssd_shared_prefix_attention(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), INVALID), (dict(pages=None), INVALID), (dict(out=None), INVALID), (dict(tables=None), INVALID),
    (dict(seq_lens=None), INVALID), (dict(starts=None), INVALID), (dict(prefixes=None), INVALID),
    (dict(dtype=2), INVALID), (dict(layer=2), INVALID), (dict(layer=-1), INVALID), (dict(hq=7), INVALID),
    (dict(groups=0), INVALID), (dict(groups=-1), INVALID), (dict(B=-1), INVALID), (dict(T=-1), INVALID),
    (dict(max_seq_len=129), INVALID), (dict(max_seq_len=0), INVALID), (dict(block_size=0), INVALID),
    (dict(D=96), UNSUPPORTED), (dict(q=P + 8), UNSUPPORTED), (dict(pages=P + 2), UNSUPPORTED),
    (dict(out=P + 4), UNSUPPORTED), (dict(B=1025), UNSUPPORTED), (dict(groups=1025), UNSUPPORTED),
    (dict(num_blocks=1 << 28), UNSUPPORTED), (dict(), WORKSPACE), (dict(ws=None, ws_bytes=1 << 30), WORKSPACE),
    (dict(ws=P + 8, ws_bytes=1 << 40), UNSUPPORTED), (dict(B=0), OK), (dict(T=0), OK)])
def test_attention_refusals(kw, rc):
    assert attention(**kw) == rc


def test_attention_workspace():
    size = lib().ssd_shared_prefix_attention_workspace_size
    assert size(0, 4, 1, 8, 1, 256, 16, 1, 4096) > 0
    for bad in ((2, 4, 1, 8, 1, 256, 16, 1, 4096), (0, 0, 1, 8, 1, 256, 16, 1, 4096), (0, 4, 1, 8, 3, 256, 16, 1, 4096),
                (0, 4, 1, 8, 1, 256, 0, 1, 4096), (0, 4, 1, 8, 1, 256, 16, 0, 4096), (0, 4, 1, 8, 1, 256, 16, 1, 0)):
        assert size(*bad) == 0


def select(**kw):
    a = dict(stream=None, logits=P, ld=1000, scores=P, lengths=P, finished=P, eos=1, alpha=0.5, o_s=P, o_p=P, o_t=P,
             o_l=P, o_f=P, ws=P, ws_bytes=0, G=2, W=4, V=1000)
    a.update(kw)
    return lib().ssd_beam_select(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(logits=None), INVALID), (dict(scores=None), INVALID), (dict(o_s=None), INVALID), (dict(o_p=None), INVALID),
    (dict(o_t=None), INVALID), (dict(ld=999), INVALID), (dict(eos=1000), INVALID), (dict(eos=-2), INVALID),
    (dict(eos=-1), INVALID), (dict(alpha=float("nan")), INVALID), (dict(lengths=None), INVALID), (dict(W=0), INVALID),
    (dict(V=0, ld=0, eos=-1, finished=None), INVALID), (dict(G=-1), INVALID), (dict(W=33), UNSUPPORTED),
    (dict(G=16384), UNSUPPORTED), (dict(V=1 << 27, ld=1 << 27), UNSUPPORTED), (dict(), WORKSPACE),
    (dict(ws=P + 4, ws_bytes=1 << 40), UNSUPPORTED), (dict(G=0), OK)])
def test_select_refusals(kw, rc):
    assert select(**kw) == rc


def test_select_workspace():
    size = lib().ssd_beam_select_workspace_size
    assert size(2, 4, 256000) > 0 and size(0, 4, 10) == 0 and size(2, 33, 10) == 0 and size(2, 4, 0) == 0


def reorder(**kw):
    a = dict(stream=None, tables=P, lens=P, max_blocks=8, free=P, top=P, refs=P, num_blocks=64, parents=P, held=P, bs=16,
             ok=None, src=P, dst=P, rows=P, G=2, W=4)
    a.update(kw)
    return lib().ssd_page_reorder(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(G=0), OK)] + [(dict([(k, None)]), INVALID) for k in (
    "tables", "lens", "free", "top", "refs", "parents", "held", "src", "dst", "rows")] + [
    (dict(W=0), INVALID), (dict(G=-1), INVALID), (dict(bs=0), INVALID), (dict(max_blocks=0), INVALID),
    (dict(num_blocks=0), INVALID), (dict(G=257), UNSUPPORTED), (dict(G=1, W=33), UNSUPPORTED), (dict(num_blocks=1 << 30), UNSUPPORTED)])
def test_reorder_refusals(kw, rc):
    assert reorder(**kw) == rc


def copy_rows(**kw):
    a = dict(stream=None, pages=P, scales=None, num_blocks=64, bs=16, planes=4, row_bytes=128, per=0, src=P, dst=P,
             rows=P, n=3)
    a.update(kw)
    return lib().ssd_page_copy_rows(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(n=0), OK), (dict(pages=None), INVALID), (dict(src=None), INVALID), (dict(dst=None), INVALID),
    (dict(rows=None), INVALID), (dict(per=2), INVALID), (dict(per=-1), INVALID), (dict(n=-1), INVALID),
    (dict(row_bytes=0), INVALID), (dict(planes=0), INVALID), (dict(row_bytes=(1 << 27) + 1), UNSUPPORTED),
    (dict(planes=65536), UNSUPPORTED)])
def test_copy_rows_refusals(kw, rc):
    assert copy_rows(**kw) == rc


def test_oracle_select_known_answer():
    x = np.log(np.array([[[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]], np.float32))
    s, p, t, n, f = beams.beam_select(x, np.log(np.array([[0.6, 0.4]])), np.array([[1, 1]]), None, 2, 0.0)
    assert p.tolist() == [[1, 0]] and t.tolist() == [[2, 0]] and f.tolist() == [[1, 0]] and n.tolist() == [[2, 2]]
    assert np.allclose(np.exp(s), [[0.32, 0.3]])
    s, p, t, n, f = beams.beam_select(x, np.log(np.array([[0.6, 0.4]])), np.array([[1, 1]]), np.array([[1, 0]]), 2, 1.0)
    # the finished beam stays at log 0.6 over one token, beam 1's best is log 0.32 over two
    assert p.tolist() == [[0, 1]] and t.tolist() == [[2, 2]] and n.tolist() == [[1, 2]]


def test_oracle_reorder_known_answer():
    # two rows of 20 tokens, block 0 shared, blocks 1 and 2 their own; both children of row 1
    new, refs, free, ok, copies = beams.reorder([[0, 1], [0, 2]], [2, 2], {0: 2, 1: 1, 2: 1}, [7], np.array([[1, 1]]),
                                                [20, 20], 16)
    assert new == [[0, 2], [0, 1]] and refs == {0: 2, 1: 1, 2: 1} and free == [7] and copies == [(1, 2, 1, 4)] and ok == [1, 1]


def test_oracle_attention_equals_plain_attention():
    rng = np.random.default_rng(0)
    pages = rng.standard_normal((2, 6, 4, 1, 8))
    tables = np.array([[3, 1, 0], [3, 2, 5]])
    q = rng.standard_normal((2, 1, 2, 8))
    out, _, _ = beams.prefix_attention(q, pages, tables, np.array([9, 11]), None, [0, 2], [4], 0.5)
    for b, n in enumerate((9, 11)):
        k, v = (pages[x, tables[b]].reshape(12, 8)[:n] for x in (0, 1))
        w = np.exp(q[b, 0] @ k.T * 0.5)
        assert np.allclose(out[b, 0], w @ v / w.sum(1, keepdims=True))


def test_polls_below_the_default_mark_are_refused():
    assert lib().ssd_shared_prefix_attention_set_polls(-2) == INVALID
    assert lib().ssd_shared_prefix_attention_set_polls(-1) == OK
