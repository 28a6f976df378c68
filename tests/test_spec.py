"""Trees of drafted tokens on the CPU: masks from parents, the calls' refusals (before any device
work), and the reference walk itself, whose accepted tokens are distributed as the target's."""
import ctypes as C

import numpy as np
import pytest

from spec_ref import ancestors, make_tree, mask_words, target, verify

EINVAL, ESCRATCH = -1, -6
A16 = C.c_void_p(1 << 20)  # an aligned address that a refused call never reads


@pytest.mark.parametrize("n,width", [(1, 1), (2, 1), (63, 2), (64, 1), (65, 3), (256, 4)])
def test_tree_masks(pkg, n, width):
    parent = make_tree(np.random.default_rng(n), n, width)
    assert np.array_equal(pkg.tree_masks(parent), mask_words(ancestors(parent)))


@pytest.mark.parametrize("parent", [[0], [-1, 1], [-1, -1], [-1, 0, 2], [-1] + list(range(256))])
def test_tree_masks_refuses_what_is_no_tree(pkg, parent):
    with pytest.raises(RuntimeError, match="-1"):
        pkg.tree_masks(parent)


def attn(pkg, **kw):
    a = dict(device=0, kv=0, q=A16, ldq=256, k=A16, v=A16, masks=A16, n=4, h=4, g=2, hd=64, past=10, seq=20, layout=0,
             out=A16, ldo=256, ws=A16, ws_bytes=1 << 30, stream=None)
    a.update(kw)
    return pkg.hip_lib().tf_hip_attn_tree(*a.values())


BAD_ATTN = [dict(kv=2), dict(kv=-1), dict(q=None), dict(k=None), dict(v=None), dict(masks=None), dict(out=None),
            dict(ldq=255), dict(ldo=255), dict(n=0), dict(n=257, seq=1000), dict(h=3), dict(h=0), dict(g=0), dict(g=-2),
            dict(h=1026, ldq=1 << 20, ldo=1 << 20), dict(hd=0), dict(hd=12), dict(hd=264, ldq=2000, ldo=2000),
            dict(hd=-8), dict(past=-1), dict(past=17), dict(past=2**31 - 2, seq=2**31 - 1), dict(layout=2),
            dict(layout=-1), dict(k=C.c_void_p((1 << 20) + 8)), dict(v=C.c_void_p((1 << 20) + 4)),
            dict(q=C.c_void_p((1 << 20) + 2)), dict(masks=C.c_void_p((1 << 20) + 4)),
            dict(ws=C.c_void_p((1 << 20) + 8))]


@pytest.mark.parametrize("bad", BAD_ATTN, ids=str)
def test_attn_tree_refusals(pkg, bad):
    assert attn(pkg, **bad) == EINVAL


def test_attn_tree_workspace(pkg):
    ws = pkg.hip_lib().tf_hip_attn_tree_ws
    need = ws(4, 4, 2, 64, 1000)
    assert need > 0
    assert attn(pkg, past=1000, seq=2000, ws_bytes=need - 1) == ESCRATCH
    assert attn(pkg, past=1000, seq=2000, ws=None, ws_bytes=0) == ESCRATCH
    for bad in ((0, 4, 2, 64, 0), (257, 4, 2, 64, 0), (4, 3, 2, 64, 0), (4, 4, 2, 60, 0), (4, 4, 2, 64, -1),
                (4, 4, 0, 64, 0), (4, 4, 2, 64, 2**31 - 1)):
        assert ws(*bad) == EINVAL


def ver(pkg, **kw):
    a = dict(device=0, logits=A16, ld=1000, vocab=1000, tokens=A16, parent=A16, n=4, draft=None, ldd=0, temperature=1.0,
             top_p=1.0, draws=A16, path=A16, result=A16, probs=None, ws=A16, ws_bytes=1 << 30, stream=None)
    a.update(kw)
    return pkg.hip_lib().tf_hip_verify_tree(*a.values())


BAD_VERIFY = [dict(logits=None), dict(ld=999), dict(vocab=0), dict(vocab=(1 << 19) + 1, ld=1 << 20), dict(tokens=None),
              dict(parent=None), dict(n=0), dict(n=257), dict(draft=A16, ldd=999), dict(temperature=float("nan")),
              dict(temperature=float("inf")), dict(top_p=float("nan")), dict(draws=None), dict(path=None),
              dict(result=None), dict(logits=C.c_void_p((1 << 20) + 2)), dict(ws=C.c_void_p((1 << 20) + 4))]


@pytest.mark.parametrize("bad", BAD_VERIFY, ids=str)
def test_verify_tree_refusals(pkg, bad):
    assert ver(pkg, **bad) == EINVAL


def test_verify_tree_workspace(pkg):
    ws = pkg.hip_lib().tf_hip_verify_tree_ws
    need = ws(4, 1000)
    assert need > 0
    assert ver(pkg, ws_bytes=need - 1) == ESCRATCH and ver(pkg, ws=None) == ESCRATCH
    for bad in ((0, 1000), (257, 1000), (4, 0), (4, (1 << 19) + 1)):
        assert ws(*bad) == EINVAL


def keep(pkg, **kw):
    a = dict(device=0, kv=0, k=A16, v=A16, layers=2, g=2, hd=64, past=10, n=4, seq=20, layout=0, path=A16, count=A16,
             stream=None)
    a.update(kw)
    return pkg.hip_lib().tf_hip_keep_path(*a.values())


@pytest.mark.parametrize("bad", [dict(kv=3), dict(k=None), dict(v=None), dict(layers=0), dict(g=0), dict(hd=4),
                                 dict(past=-1), dict(past=17), dict(n=0), dict(n=257, seq=1000), dict(layout=2),
                                 dict(path=None), dict(count=None), dict(k=C.c_void_p((1 << 20) + 8)),
                                 dict(path=C.c_void_p((1 << 20) + 2))], ids=str)
def test_keep_path_refusals(pkg, bad):
    assert keep(pkg, **bad) == EINVAL


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("top_p", [1.0, 0.8])
def test_reference_walk_keeps_the_target_distribution(sampled, top_p):
    """Over many draws (and, where the drafts are sampled, many drafts) the token that follows the
    settled one (the first accepted child's, else the next token) is distributed as the target. The
    counts' deviation is that of N draws: 5 sqrt(p (1 - p) / N) is passed less than once in a million."""
    rng = np.random.default_rng(12)
    vocab, n_draws = 6, 20000
    logits = rng.standard_normal((4, vocab)).astype(np.float32)
    parent = np.array([-1, 0, 0, 0], np.int32)
    q = target(logits[0] + rng.standard_normal(vocab), 1.0, 1.0)
    want = target(logits[0], 0.9, top_p)
    got = np.zeros(vocab)
    fixed = np.argsort(-q)[:3]
    for _ in range(n_draws):
        kids = rng.choice(vocab, 3, p=q) if sampled else fixed
        tokens = np.array([0, *kids], np.int32)
        path, token, _ = verify(logits, tokens, parent, np.tile(q, (4, 1)) if sampled else None, 0.9, top_p,
                                rng.random(4))
        got[tokens[path[1]] if len(path) > 1 else token] += 1
    dev = np.sqrt(want * (1 - want) / n_draws)
    assert np.all(np.abs(got / n_draws - want) <= 5 * dev + 1e-12)
