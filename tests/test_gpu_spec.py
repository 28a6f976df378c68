"""Trees of drafted tokens on the GPU (tf_hip_attn_tree, tf_hip_verify_tree, tf_hip_keep_path)
against plain forms in 64 bits, through the C ABI with device memory from torch."""
import math

import numpy as np
import pytest
import torch

from spec_ref import ancestors, make_tree, mask_words, verify

pytestmark = pytest.mark.gpu

F32, F16 = 0, 1
DEV = "cuda"
NAN = float("nan")
EPS = 2.0 ** -24  # half a step of fp32, relative


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.hip_lib()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------- attention of a tree

class Attn:
    """One call's inputs. Cache rows behind the tree hold NaN, and so do the output's columns behind a row."""

    def __init__(self, h, g, hd, n, past, slack=3, layout=0, kv=F32, mask="tree", seed=0, pad=0, shift=0):
        self.__dict__.update(h=h, g=g, hd=hd, n=n, past=past, layout=layout, kv=kv, seq=past + n + slack)
        rng = np.random.default_rng([seed, h, g, hd, n, past])
        if mask == "all":
            see = np.ones((n, n), bool)
        elif mask == "random":  # not a tree: rows that see nothing among them
            see = rng.random((n, n)) < 0.3
            see[:: 2] = False
        else:
            see = ancestors(make_tree(rng, n, 1 if mask == "chain" else 3))
        self.see = torch.from_numpy(see).to(DEV)
        words = mask_words(see)
        if n % 64:  # bits past n_tree are not looked at
            words[:, -1] |= np.uint64((~((1 << (n % 64)) - 1)) & ((1 << 64) - 1))
        self.masks = torch.from_numpy(words.view(np.int64)).to(DEV)
        gen = torch.Generator(device=DEV)
        gen.manual_seed(seed + 1000 * n + past)
        self.ld = h * hd + pad
        buf = torch.randn(n * self.ld + shift, generator=gen, device=DEV)
        self.q = buf[shift:].view(n, self.ld)
        shape = (self.seq, g, hd) if layout == 0 else (g, self.seq, hd)
        t = torch.float32 if kv == F32 else torch.float16
        self.k, self.v = (torch.randn(shape, generator=gen, device=DEV).to(t) for _ in range(2))
        for x in (self.k, self.v):
            self.rows(x)[past + n:] = NAN
        self.out = torch.full((n, self.ld), NAN, device=DEV)
        self.ws = None

    def rows(self, x):
        """A cache as [position][kv head][hd]."""
        return x if self.layout == 0 else x.transpose(0, 1)

    def call(self, lib):
        if self.ws is None:
            nb = lib.tf_hip_attn_tree_ws(self.n, self.h, self.g, self.hd, self.past)
            assert nb >= 0
            self.ws = torch.full((nb + 64,), 0xFF, dtype=torch.uint8, device=DEV)  # NaN in every word
        rc = lib.tf_hip_attn_tree(0, self.kv, self.q.data_ptr(), self.ld, self.k.data_ptr(), self.v.data_ptr(),
                                  self.masks.data_ptr(), self.n, self.h, self.g, self.hd, self.past, self.seq,
                                  self.layout, self.out.data_ptr(), self.ld, self.ws.data_ptr(), self.ws.numel() - 64,
                                  stream())
        assert rc == 0
        return self.out

    def run(self, lib):
        self.call(lib)
        torch.cuda.synchronize()
        assert bool((self.ws[-64:] == 0xFF).all()), "written past the workspace"
        w = self.h * self.hd
        assert bool(torch.isnan(self.out[:, w:]).all()), "written past a row"
        return self.out[:, :w].view(self.n, self.h, self.hd).double()

    def want(self):
        """The result in 64 bits, and what an element may be off.

        A score of hd products is off by at most e = (3 hd / 32 + 34) eps a for the additions (in steps of
        32 terms, three products each for split fp32 numbers) and 4 eps' a for the numbers' rounding to 22
        bits and the product of the two rests that is left out (eps' = 2^-22), a = sum |q k| / sqrt(hd); a
        weight e^s then by the factor 2 e, with 2^-22 for the exponential. The sums over positions take
        at most n / 8 + 64 additions one after the other, the weights and values 22 bits again, and the
        quotient doubles all of it; sum p |v| is what that multiplies."""
        n, h, hd, rep = self.n, self.h, self.hd, self.h // self.g
        end = self.past + n
        out = torch.zeros(n, h, hd, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        see = torch.cat((torch.ones(n, self.past, dtype=torch.bool, device=DEV), self.see), 1)
        for g in range(self.g):
            k = self.rows(self.k)[:end, g].double().contiguous()
            v = self.rows(self.v)[:end, g].double().contiguous()
            for head in range(g * rep, (g + 1) * rep):
                q = self.q[:, head * hd: (head + 1) * hd].double()
                s = torch.where(see, (q @ k.t().contiguous()) / math.sqrt(hd), -math.inf)
                a = torch.where(see, (q.abs() @ k.abs().t().contiguous()) / math.sqrt(hd), 0.0).amax(1)
                top = s.amax(1, keepdim=True)
                p = torch.where(see, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
                p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
                e = (3 * hd / 32 + 34) * EPS * a + 4 * 2.0 ** -22 * a
                out[:, head] = p @ v
                tol[:, head] = (p @ v.abs()) * (2 * (2 * e + 2.0 ** -22 + (end / 8 + 64) * EPS + 2.0 ** -21))[:, None]
        return out, tol

    def check(self, lib):
        got, (want, tol) = self.run(lib), self.want()
        assert not bool(torch.isnan(got).any())
        off = (got - want).abs()
        assert bool((off <= tol).all()), f"off by {float((off / tol.clamp_min(1e-30)).max()):.3g} tolerances"
        # roundings of either sign add as their squares do: the whole is nearer than the worst element
        norm = float(want.norm())
        if norm:
            assert float(off.norm()) <= 2.0 ** -17 * norm
        empty = ~self.see.any(1) if self.past == 0 else torch.zeros(self.n, dtype=torch.bool, device=DEV)
        assert bool((got[empty] == 0).all())
        return got


SHAPES = [
    # heads, kv heads, head size, nodes, past
    (4, 2, 64, 1, 0), (32, 8, 64, 1, 6), (14, 2, 64, 1, 33), (32, 8, 64, 2, 31), (32, 8, 64, 3, 32), (12, 2, 128, 4, 1),
    (12, 2, 128, 5, 63), (32, 8, 64, 8, 1000), (14, 2, 64, 37, 2029), (32, 8, 64, 16, 64), (32, 8, 64, 17, 65),
    (6, 6, 64, 33, 127), (4, 1, 128, 63, 200), (32, 8, 64, 64, 129), (14, 2, 64, 65, 95), (12, 2, 128, 100, 517),
    (32, 8, 64, 128, 3), (8, 8, 128, 129, 0), (12, 4, 64, 256, 0), (12, 2, 128, 256, 301), (48, 1, 64, 7, 260),
    (17, 1, 64, 3, 70), (5, 5, 32, 9, 41), (64, 8, 128, 64, 4100), (32, 8, 64, 1, 9000), (9, 3, 128, 11, 5003),
]


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attn_tree(lib, shape, kv, layout):
    Attn(*shape, layout=layout, kv=kv, seed=1).check(lib)


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("n", [1, 6, 40])
@pytest.mark.parametrize("hd", [8, 16, 24, 32, 40, 56, 72, 80, 96, 104, 120, 136, 160, 192, 224, 248, 256])
def test_attn_tree_head_sizes(lib, hd, n, kv):
    Attn(6, 2, hd, n, 75, kv=kv, layout=hd // 8 % 2, seed=2).check(lib)


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("past", [0, 1, 50])
@pytest.mark.parametrize("mask", ["chain", "all", "random"])
@pytest.mark.parametrize("n", [1, 7, 66])
def test_attn_tree_masks(lib, n, mask, past, kv):
    """Chains, full masks, and masks that are no tree, whose rows may see nothing (with no past: zero)."""
    Attn(8, 2, 64, n, past, mask=mask, kv=kv, seed=3).check(lib)


@pytest.mark.parametrize("h,g,hd,n,past", [(1024, 4, 8, 3, 40), (1024, 1024, 8, 2, 10), (64, 1, 64, 256, 40),
                                           (256, 1, 128, 5, 300)])
def test_attn_tree_many_heads(lib, h, g, hd, n, past):
    """Up to 1,024 query heads, over one kv head or as many: rows past one workgroup's, splits of one."""
    Attn(h, g, hd, n, past, seed=16).check(lib)


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("h,g,hd,n,past", [(8, 1, 64, 40, 16400), (6, 1, 128, 48, 16650), (9, 1, 72, 30, 17000)])
def test_attn_tree_wide_workgroups(lib, h, g, hd, n, past, kv):
    """Rows and steps enough for the workgroups of 256 rows, the last of them not full, the head size padded in
    one."""
    Attn(h, g, hd, n, past * 8, kv=kv, layout=n // 8 % 2, seed=17).check(lib)


@pytest.mark.parametrize("pad,shift", [(0, 1), (5, 0), (64, 3)])
@pytest.mark.parametrize("n", [1, 9, 70])
def test_attn_tree_strides_and_alignment(lib, n, pad, shift):
    """Queries and outputs inside wider rows (a QKV row's), at any 4-byte address."""
    Attn(4, 2, 64, n, 90, pad=pad, shift=shift, seed=4).check(lib)


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("n", [2, 24, 70])
@pytest.mark.parametrize("past", [0, 5, 64])
@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
def test_attn_tree_unseen_rows_do_not_matter(lib, bad, past, n, kv):
    """Infinities and NaN in a node's key and value rows leave the queries that do not see it as they are,
    bit for bit; they reach those that do."""
    x = Attn(8, 2, 64, n, past, kv=kv, seed=5)
    before = x.run(lib).clone()
    node = n // 2
    x.rows(x.k)[past + node] = bad
    x.rows(x.v)[past + node] = bad
    after = x.run(lib)
    blind = ~x.see[:, node]
    assert bool(blind.any()) and torch.equal(after[blind], before[blind])
    assert not bool(torch.isfinite(after[~blind]).any())


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("n", [1, 20])
def test_attn_tree_scales(lib, n, kv):
    """Rows of keys, values and queries scaled by powers of two from 2^-8 to 2^8 (keys and queries against
    each other), values that are zero, and values of another size in another part of the cache."""
    x = Attn(8, 2, 64, n, 300, kv=kv, seed=6)
    e = torch.arange(303 + n, device=DEV) % 17 - 8
    f = torch.exp2(e.float()).to(x.k.dtype)[: x.seq]
    x.rows(x.v).mul_(f[:, None, None])
    x.rows(x.v)[10:20] = 0.0
    x.rows(x.v)[100:180] *= 2.0 ** -6
    x.rows(x.k).mul_(2.0 ** -7 if kv == F16 else 2.0 ** -30)
    x.q.mul_(2.0 ** 7 if kv == F16 else 2.0 ** 30)
    got, (want, tol) = x.run(lib), x.want()
    assert bool(((got - want).abs() <= tol).all())


def test_attn_tree_values_of_zero_and_sharp_rows(lib):
    """All values zero: zero. Queries that leave one position all the weight: that position's value."""
    x = Attn(4, 2, 64, 5, 100, seed=7)
    x.v[: 105] = 0.0
    assert bool((x.run(lib) == 0).all())
    x = Attn(4, 2, 64, 5, 100, seed=8)
    x.q.copy_(64.0 * x.rows(x.k)[17].repeat_interleave(2, 0).reshape(1, -1))
    got = x.check(lib)
    want = x.rows(x.v)[17].repeat_interleave(2, 0).double()
    assert float((got - want).abs().max()) < 1e-5


def test_attn_tree_one_query_is_decode_attention(lib, pkg):
    """n_tree = 1 over the rows of tf_hip_attn_decode: within the two kernels' tolerances of each other."""
    x = Attn(32, 8, 64, 1, 700, seed=9)
    got, (_, tol) = x.run(lib), x.want()
    rows = [x.rows(c)[:701].cpu().numpy() for c in (x.k, x.v)]
    want = torch.from_numpy(pkg.attn_decode(x.q.view(32, 64).cpu().numpy(), *rows, 1024, 0)).to(DEV).double()
    assert bool(((got[0] - want).abs() <= 2 * tol[0]).all())


@pytest.mark.parametrize("layout", [0, 1])
def test_attn_tree_offsets_past_32_bits(lib, layout):
    """A cache of more than 2^32 bytes and 2^31 elements, read at its end."""
    g, hd, seq = 8, 128, 2_400_000
    k, v = (torch.zeros((seq, g, hd) if layout == 0 else (g, seq, hd), dtype=torch.float16, device=DEV)
            for _ in range(2))
    assert k.numel() > 2**31
    x = Attn(8, g, hd, 3, 200, slack=0, kv=F16, seed=10)
    if layout == 0:  # a long context of equal keys and values, then the last rows
        past = seq - 3
        v.fill_(0.25)
        rows = k[-3:], v[-3:]
    else:
        past = 200
        rows = k[:, :203].transpose(0, 1), v[:, :203].transpose(0, 1)
    rows[0].copy_(x.k[-rows[0].shape[0]:])
    rows[1].copy_(x.v[-rows[1].shape[0]:])
    small = x.want()[0] if layout else None
    x.k, x.v, x.layout, x.seq, x.past = k, v, layout, seq, past
    got = x.run(lib)
    if layout == 0:
        # past keys are zero: weight 1 each, value 0.25; the tree's rows weigh e^s
        q = x.q.view(3, g, hd).double()
        s = torch.einsum("ngd,jgd->ngj", q.cpu(), k[-3:].double().cpu()).to(DEV) / math.sqrt(hd)
        w = torch.where(x.see[:, None, :], torch.exp(s), 0.0)
        num = 0.25 * past + torch.einsum("ngj,jgd->ngd", w.cpu(), v[-3:].double().cpu()).to(DEV)
        want = num / (past + w.sum(2, keepdim=True))
        # 2.4 million equal terms: (past / 8 + 64) additions at the most, as in want(), but all of one sign
        # and value; the mean of equal values is off by far less
        assert float((got - want).abs().max()) < 1e-5
    else:
        assert float((got - small).abs().max()) < 1e-5


def test_attn_tree_on_streams_and_in_graphs(lib):
    """Two calls at once on streams of their own with workspaces of their own; then one captured into a
    graph and replayed with eager calls and new inputs between, each replay checked."""
    xs = [Attn(32, 8, 64, n, 600, seed=11 + n) for n in (8, 64)]
    want = [x.check(lib).clone() for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for x in xs:
        x.out.fill_(NAN)
    torch.cuda.synchronize()
    for _ in range(10):
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                x.call(lib)
    torch.cuda.synchronize()
    for x, w in zip(xs, want):
        assert torch.equal(x.out.view(x.n, x.h, x.hd).double(), w)
    x, other = xs
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.call(lib)
    for i in range(4):
        x.q.copy_(torch.randn_like(x.q))
        x.out.fill_(NAN)
        graph.replay()
        got = x.out.clone()
        other.call(lib)
        assert torch.equal(x.call(lib), got), i
        x.check(lib)


def test_attn_tree_is_deterministic(lib):
    x = Attn(32, 8, 64, 29, 3000, seed=12)
    a = x.run(lib).clone()
    for _ in range(3):
        assert torch.equal(x.run(lib), a)


# ---------------------------------------------------------------- verification

class Verify:
    def __init__(self, n, vocab, width=1, sampled=False, scale=4.0, temperature=0.8, top_p=1.0, seed=0, pad=0, shift=0):
        self.__dict__.update(n=n, vocab=vocab, sampled=sampled, temperature=temperature, top_p=top_p, pad=pad,
                             shift=shift)
        rng = np.random.default_rng([seed, n, vocab, width])
        self.parent = make_tree(rng, n, width)
        self.logits = (scale * rng.standard_normal((n, vocab))).astype(np.float32)
        drafted = self.logits + 0.2 * scale * rng.standard_normal((n, vocab)).astype(np.float32)
        self.draft = None
        self.tokens = rng.integers(0, vocab, n).astype(np.int32)
        seen = {}
        for i in range(1, n):
            p = int(self.parent[i])
            k = seen.get(p, 0)
            seen[p] = k + 1
            if not sampled:
                self.tokens[i] = np.argsort(-drafted[p])[min(k, vocab - 1)]
        if sampled:
            d = np.exp((drafted - drafted.max(1, keepdims=True)) / (temperature or 1.0)).astype(np.float64)
            self.draft = (d / d.sum(1, keepdims=True)).astype(np.float32)
            for i in range(1, n):
                cum = np.cumsum(self.draft[self.parent[i]].astype(np.float64))
                self.tokens[i] = min(int(np.searchsorted(cum, rng.random() * cum[-1])), vocab - 1)
        self.draws = rng.random(n).astype(np.float32)

    def rows(self, a):
        """Rows `pad` apart more than they are long, `shift` floats into an allocation."""
        n, v = a.shape
        buf = torch.full((self.shift + n * (v + self.pad),), NAN, device=DEV)
        t = buf[self.shift:].view(n, v + self.pad)
        t[:, :v] = torch.from_numpy(a)
        return t

    def setup(self, lib):
        n = self.n
        up = lambda a: torch.from_numpy(a).to(DEV)  # noqa: E731
        self.d = dict(logits=self.rows(self.logits), draft=None if self.draft is None else self.rows(self.draft),
                      tokens=up(self.tokens), parent=up(self.parent), draws=up(self.draws),
                      path=torch.full((n + 1,), -77, dtype=torch.int32, device=DEV),
                      result=torch.full((3,), -77, dtype=torch.int32, device=DEV),
                      probs=torch.full((n + 1,), -77.0, device=DEV))
        nb = lib.tf_hip_verify_tree_ws(n, self.vocab)
        self.ws = torch.full((nb + 64,), 0xFF, dtype=torch.uint8, device=DEV)
        return self

    def call(self, lib, probs=True):
        d, ld = self.d, self.vocab + self.pad
        rc = lib.tf_hip_verify_tree(0, d["logits"].data_ptr(), ld, self.vocab, d["tokens"].data_ptr(),
                                    d["parent"].data_ptr(), self.n,
                                    None if d["draft"] is None else d["draft"].data_ptr(), ld, self.temperature,
                                    self.top_p, d["draws"].data_ptr(), d["path"].data_ptr(), d["result"].data_ptr(),
                                    d["probs"].data_ptr() if probs else None, self.ws.data_ptr(), self.ws.numel() - 64,
                                    stream())
        assert rc == 0

    def read(self):
        torch.cuda.synchronize()
        assert bool((self.ws[-64:] == 0xFF).all()), "written past the workspace"
        d = self.d
        assert int(d["path"][-1]) == -77 and int(d["result"][-1]) == -77 and float(d["probs"][-1]) == -77.0
        return d["path"][:-1].cpu().numpy(), d["result"][:-1].tolist(), d["probs"][:-1].cpu().numpy()

    def check(self, lib):
        self.setup(lib).call(lib)
        got_path, (count, token), got_probs = self.read()
        path, want_token, probs = verify(self.logits, self.tokens, self.parent, self.draft, self.temperature, self.top_p,
                                         self.draws)
        assert count == len(path) and got_path.tolist() == path + [-1] * (self.n - count)
        assert token == want_token
        # a probability's numerator is a 64-bit exponential; its row's sum has terms that are each off by
        # the difference's rounding times the exponent (at most 24 of them count) and the exponential's
        # own 2 steps: 2^-24 (24 + 4) at the worst, and the rounding to fp32
        assert np.all(np.abs(got_probs - probs) <= (2.0 ** -24 * 30) * probs + 1e-37)
        return path, token


CASES = [(1, 7, 1), (2, 64, 1), (5, 1000, 1), (6, 32000, 2), (16, 4096, 3), (40, 999, 4), (64, 2049, 4), (65, 300, 2),
         (256, 50, 3), (5, 128256, 1), (3, 151936, 2), (2, 524288, 1)]


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("temperature,top_p", [(0.0, 1.0), (0.8, 1.0), (1.3, 0.9), (0.7, 0.3)])
@pytest.mark.parametrize("n,vocab,width", CASES)
def test_verify_tree(lib, n, vocab, width, temperature, top_p, sampled):
    for seed in range(2 if n * vocab > 100000 else 6):
        Verify(n, vocab, width, sampled, temperature=temperature, top_p=top_p, seed=seed).check(lib)


@pytest.mark.parametrize("scale", [0.001, 0.05, 1.0, 30.0, 1000.0])
@pytest.mark.parametrize("top_p", [0.0, 1e-6, 0.37, 0.96, 0.99999, 1.0])
def test_verify_tree_flat_and_sharp(lib, scale, top_p):
    """From distributions over the whole vocabulary to ones of a single token."""
    for seed in range(3):
        Verify(4, 20011, 2, seed == 2, scale=scale, temperature=0.9, top_p=top_p, seed=20 + seed).check(lib)


@pytest.mark.parametrize("top_p", [0.31, 0.93, 1.0])
@pytest.mark.parametrize("steps", [1, 3, 40])
@pytest.mark.parametrize("vocab", [999, 9001, 100003])
def test_verify_tree_ties(lib, vocab, steps, top_p):
    """Logits of few values (steps = 1: all equal), so that the nucleus ends among equal ones; more of them
    than one list holds. The sums of equal weights are exact on both sides, and top_p (a rounded number)
    falls between two of them."""
    for seed in range(4):
        x = Verify(6, vocab, 2, seed % 2 == 1, temperature=0.7, top_p=top_p, seed=30 + seed)
        x.logits = (np.floor(x.logits / 30 * steps) * (3.0 / steps)).astype(np.float32)
        if steps == 1:
            x.logits[:] = 2.5
        x.check(lib)


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("top_p", [0.4, 1.0])
@pytest.mark.parametrize("vocab", [1, 2, 3, 17])
def test_verify_tree_small_vocabularies(lib, vocab, top_p, sampled):
    """Down to one token, with more siblings than tokens."""
    for seed in range(8):
        Verify(9, vocab, 4, sampled, scale=1.0, top_p=top_p, seed=100 + seed).check(lib)


@pytest.mark.parametrize("top_p", [0.2, 0.77, 0.999])
def test_verify_tree_crowded_bins(lib, top_p):
    """One far logit stretches the row's range, so that tens of thousands of others, all different, share a bin;
    and rows whose nucleus ends in the last bin, 24 temperatures down and further."""
    for seed in range(3):
        x = Verify(4, 60001, 2, False, scale=0.001, temperature=0.9, top_p=top_p, seed=110 + seed)
        x.logits[:, 7] = -15.0
        x.logits[1] = np.where(np.arange(60001) == 99, 26.0, x.logits[1]).astype(np.float32)
        x.check(lib)


@pytest.mark.parametrize("n,vocab,kw", [
    (64, 4097, dict(seed=8001, width=2, scale=3.0, temperature=2.0, top_p=0.99, pad=5, shift=3)),
    (16, 8192, dict(seed=1497, width=2, sampled=True, scale=1.0, temperature=1.0, top_p=0.5, pad=1))])
def test_verify_tree_nucleus_border(lib, n, vocab, kw):
    """A row's running sum passes top_p by 5e-10 and 4e-9: sums of 32-bit weights keep another last token."""
    Verify(n, vocab, **kw).check(lib)


def test_verify_tree_many_rejections(lib):
    """Nodes with up to 40 children sampled from a distribution far from the target's, so that most are rejected
    and one sum over the row follows another."""
    for seed in range(6):
        x = Verify(60, 3001, 40, True, scale=2.0, top_p=(1.0, 0.9)[seed % 2], seed=120 + seed)
        rng = np.random.default_rng(seed)
        d = np.exp(2.0 * rng.standard_normal((60, 3001)))
        x.draft = (d / d.sum(1, keepdims=True)).astype(np.float32)
        for i in range(1, 60):
            cum = np.cumsum(x.draft[x.parent[i]].astype(np.float64))
            x.tokens[i] = min(int(np.searchsorted(cum, rng.random() * cum[-1])), 3000)
        x.draws[1:] = 0.5 + 0.5 * x.draws[1:]
        x.check(lib)


@pytest.mark.parametrize("top_p", [0.9, 1.0])
@pytest.mark.parametrize("sampled", [False, True])
def test_verify_tree_masked_logits(lib, sampled, top_p):
    """Logits of -inf and NaN weigh nothing, the type's lowest value hardly anything; a row of -inf alone is
    uniform; one infinite logit takes it all."""
    for seed in range(4):
        x = Verify(6, 5000, 2, sampled, top_p=top_p, seed=40 + seed)
        rng = np.random.default_rng(seed)
        for i, value in enumerate((-np.inf, np.nan, np.finfo(np.float32).min)):
            x.logits[i][rng.random(5000) < 0.7] = value
        x.logits[3] = -np.inf
        x.logits[4][123] = np.inf
        x.check(lib)


@pytest.mark.parametrize("sampled", [False, True])
def test_verify_tree_strange_trees(lib, sampled):
    """Siblings of one token, parents that are none, tokens outside the vocabulary."""
    for seed in range(6):
        x = Verify(12, 40, 4, sampled, scale=1.0, seed=50 + seed)
        x.tokens[3], x.tokens[5] = x.tokens[2], x.tokens[1]
        x.parent[2:6] = 0
        x.parent[6], x.parent[7], x.parent[8] = -1, 7, 99
        x.tokens[9], x.tokens[10] = -1, 40
        x.check(lib)


def test_verify_tree_draw_edges(lib):
    """A draw of 0 accepts whatever has any probability; one next to 1 only what is certain, and takes the
    last token that is left."""
    x = Verify(6, 300, 1, seed=60)
    x.draws[:] = 0.0
    path, _ = x.check(lib)
    assert len(path) == 6
    x.draws[:] = np.nextafter(np.float32(1), np.float32(0))
    x.check(lib)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 2), (64, 3)])
@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("vocab", [5, 4097])
def test_verify_tree_strides_and_alignment(lib, vocab, sampled, pad, shift):
    for top_p in (0.8, 1.0):
        Verify(7, vocab, 3, sampled, top_p=top_p, seed=70, pad=pad, shift=shift).check(lib)


def test_verify_tree_first_token_is_sample_logits(lib, pkg):
    """One node, temperature 0: tf_hip_argmax's token; and no output of probabilities on request."""
    x = Verify(1, 5000, temperature=0.0, seed=80).setup(lib)
    x.d["probs"].fill_(-77.0)
    x.call(lib, probs=False)
    path, (count, token), probs = x.read()
    assert count == 1 and token == pkg.argmax(x.logits[0]) and np.all(probs == -77.0)


def test_verify_tree_in_graphs_and_on_streams(lib):
    """Captured once, replayed with new logits, drafts, trees and draws, eager calls of another size between."""
    x = Verify(16, 6000, 3, True, top_p=0.9, seed=90).setup(lib)
    other = Verify(5, 9000, 1, seed=91).setup(lib)
    x.call(lib)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.call(lib)
    side = torch.cuda.Stream()
    for seed in range(92, 97):
        new = Verify(16, 6000, 3, True, top_p=0.9, seed=seed).setup(lib)
        for k in ("logits", "draft", "tokens", "parent", "draws"):
            x.d[k].copy_(new.d[k])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other.call(lib)
        graph.replay()
        other.call(lib) if seed % 2 else None
        path, (count, token), _ = x.read()
        want_path, want_token, _ = verify(new.logits, new.tokens, new.parent, new.draft, 0.8, 0.9, new.draws)
        assert path.tolist() == want_path + [-1] * (16 - count) and token == want_token


# ---------------------------------------------------------------- keeping the path

@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("layers,g,hd,past,n,slack,path", [
    (1, 1, 8, 0, 1, 0, [0]), (2, 2, 64, 0, 5, 0, [0, 1, 2, 3, 4]), (3, 2, 64, 7, 9, 2, [0, 3, 4, 8]),
    (16, 8, 64, 100, 64, 5, [0, 2, 3, 10, 11, 12, 40, 63]), (2, 3, 136, 33, 256, 1, list(range(0, 256, 2))),
    (28, 2, 128, 50, 30, 0, [0, 29]), (2, 1, 24, 4, 6, 3, []), (2, 2, 64, 9, 17, 0, [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 16]),
])
def test_keep_path(lib, layers, g, hd, past, n, slack, path, kv, layout):
    seq = past + n + slack
    shape = (layers, seq, g, hd) if layout == 0 else (layers, g, seq, hd)
    t = torch.float32 if kv == F32 else torch.float16
    k, v = (torch.randn(shape, device=DEV).to(t) for _ in range(2))
    want = []
    for x in (k, v):
        w = x.clone()
        a, b = (w, x.clone()) if layout == 0 else (w.transpose(1, 2), x.clone().transpose(1, 2))
        for i, node in enumerate(path):
            a[:, past + i] = b[:, past + node]
        want.append(w)
    p = torch.tensor(path + [-1] * (n - len(path)), dtype=torch.int32, device=DEV)
    count = torch.tensor([len(path)], dtype=torch.int32, device=DEV)
    assert lib.tf_hip_keep_path(0, kv, k.data_ptr(), v.data_ptr(), layers, g, hd, past, n, seq, layout, p.data_ptr(),
                                count.data_ptr(), stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("path,count,good", [([0, 2, 2, 3], 4, 2), ([0, 3, 1, 4], 4, 2), ([0, 2, 6, 7], 4, 2),
                                             ([0, -5, 2, 3], 4, 1), ([-1, 0, 1, 2], 4, 0), ([0, 2, 4, 5], -3, 0),
                                             ([0, 2, 4, 5, 5, 5], 1000, 4)])
def test_keep_path_ends_at_a_bad_entry(lib, path, count, good):
    """Entries that do not ascend or are no node end the path; so does its length."""
    k = torch.randn(2, 20, 2, 16, device=DEV)
    v = torch.randn_like(k)
    want = [x.clone() for x in (k, v)]
    for w, x in zip(want, (k, v)):
        for i in range(good):
            w[:, 10 + i] = x[:, 10 + path[i]]
    p = torch.tensor((path + [9] * 6)[:6], dtype=torch.int32, device=DEV)
    c = torch.tensor([count], dtype=torch.int32, device=DEV)
    assert lib.tf_hip_keep_path(0, F32, k.data_ptr(), v.data_ptr(), 2, 2, 16, 10, 6, 20, 0, p.data_ptr(), c.data_ptr(),
                                stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


# ---------------------------------------------------------------- the calls together

@pytest.mark.parametrize("layout", [0, 1])
def test_speculative_steps_match_decoding_one_by_one(lib, pkg, layout):
    """Greedy decoding of a small attention-only model (two layers, each the attention of an embedding's
    projections over the cache, with the rest of the sum added; the logits are against the embedding),
    once token by token (one-node trees) and once with trees of drafted tokens, of which some are right:
    the same tokens, and in the end the same cache rows, to the attention's rounding."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    h, g, hd, vocab, layers, seq = 4, 2, 32, 211, 2, 96
    d = h * hd
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    embed = randn(vocab, d)
    wq, wk, wv = randn(layers, d, d) / d**0.5, randn(layers, d, g * hd) / d**0.5, randn(layers, d, g * hd) / d**0.5
    place = 0.3 * randn(seq, d)  # added by position
    shape = (layers, seq, g, hd) if layout == 0 else (layers, g, seq, hd)

    class State:
        def __init__(self):
            self.k, self.v, self.past = torch.zeros(shape, device=DEV), torch.zeros(shape, device=DEV), 0

        def step(self, tokens, parent):
            """Logits after every node; the nodes' rows go into the caches behind the settled ones."""
            n = len(tokens)
            see = ancestors(parent)
            depth = see.sum(1) - 1
            x = embed[torch.tensor(tokens, device=DEV)] + place[torch.tensor(self.past + depth, device=DEV)]
            masks = torch.from_numpy(pkg.tree_masks(parent).view(np.int64)).to(DEV)
            ws = torch.empty(lib.tf_hip_attn_tree_ws(n, h, g, hd, self.past) + 16, dtype=torch.uint8, device=DEV)
            for i in range(layers):
                for cache, w in ((self.k, wk), (self.v, wv)):
                    rows = cache[i] if layout == 0 else cache[i].transpose(0, 1)
                    rows[self.past: self.past + n] = (x @ w[i]).view(n, g, hd)
                q, out = (x @ wq[i]).contiguous(), torch.empty(n, d, device=DEV)
                assert lib.tf_hip_attn_tree(0, F32, q.data_ptr(), d, self.k[i].data_ptr(), self.v[i].data_ptr(),
                                            masks.data_ptr(), n, h, g, hd, self.past, seq, layout, out.data_ptr(), d,
                                            ws.data_ptr(), ws.numel(), stream()) == 0
                x = x + out
            return (x @ embed.t().contiguous()).contiguous()

        def verify(self, logits, tokens, parent):
            n = len(tokens)
            up = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)  # noqa: E731
            tok, par, path, result = up(tokens), up(parent), up([0] * n), up([0, 0])
            draws = torch.rand(n, device=DEV)
            ws = torch.empty(lib.tf_hip_verify_tree_ws(n, vocab), dtype=torch.uint8, device=DEV)
            assert lib.tf_hip_verify_tree(0, logits.data_ptr(), vocab, vocab, tok.data_ptr(), par.data_ptr(), n, None, 0,
                                          0.0, 1.0, draws.data_ptr(), path.data_ptr(), result.data_ptr(), None,
                                          ws.data_ptr(), ws.numel(), stream()) == 0
            assert lib.tf_hip_keep_path(0, F32, self.k.data_ptr(), self.v.data_ptr(), layers, g, hd, self.past, n, seq,
                                        layout, path.data_ptr(), result.data_ptr(), stream()) == 0
            count, token = result.tolist()
            self.past += count
            return [int(tokens[i]) for i in path.tolist()[1:count]], token

    one, ids = State(), [3]
    while len(ids) < 61:
        _, token = one.verify(one.step([ids[-1]], np.array([-1], np.int32)), [ids[-1]], [-1])
        ids.append(token)
    rng = np.random.default_rng(1)
    many, got, steps = State(), [3], 0
    while len(got) < 61:
        n = int(rng.integers(2, 14))
        parent = make_tree(rng, n, 3)
        depth = ancestors(parent).sum(1) - 1
        tokens = [got[-1]]
        for i in range(1, n):  # two thirds of the drafts are what the model would say there
            at = len(got) - 1 + int(depth[i])
            tokens.append(ids[at] if rng.random() < 0.67 and at < len(ids) else int(rng.integers(vocab)))
        if many.past + n > seq:
            break
        kept, token = many.verify(many.step(tokens, parent), tokens, parent)
        got += kept + [token]
        steps += 1
    m = min(len(ids), len(got))
    assert m > 40 and got[:m] == ids[:m] and steps < len(got) - 1
    rows = min(one.past, many.past)
    for a, b in ((one.k, many.k), (one.v, many.v)):
        a, b = ((x if layout == 0 else x.transpose(1, 2))[:, :rows] for x in (a, b))
        assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max())


def test_current_device_and_default_stream(lib):
    """The calls leave the current device alone, and take the null stream."""
    x = Attn(4, 2, 64, 3, 20, seed=13)
    nb = lib.tf_hip_attn_tree_ws(3, 4, 2, 64, 20)
    ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    before = torch.cuda.current_device()
    assert lib.tf_hip_attn_tree(0, F32, x.q.data_ptr(), x.ld, x.k.data_ptr(), x.v.data_ptr(), x.masks.data_ptr(), 3, 4,
                                2, 64, 20, x.seq, 0, x.out.data_ptr(), x.ld, ws.data_ptr(), ws.numel(), None) == 0
    torch.cuda.synchronize()
    assert torch.cuda.current_device() == before
    assert lib.tf_hip_attn_tree(99, F32, x.q.data_ptr(), x.ld, x.k.data_ptr(), x.v.data_ptr(), x.masks.data_ptr(), 3, 4,
                                2, 64, 20, x.seq, 0, x.out.data_ptr(), x.ld, ws.data_ptr(), ws.numel(), None) == -4
    assert torch.cuda.current_device() == before


def test_errors_do_not_outlive_their_call(lib, pkg):
    """A call that fails (a device that is not there) leaves no error behind for the next call to find, and an
    error that another call left behind is not taken for this one's."""
    import ctypes as C
    x = Attn(4, 2, 64, 3, 20, seed=14)
    ok = x.check(lib).clone()

    def bad():
        return lib.tf_hip_attn_tree(99, F32, x.q.data_ptr(), x.ld, x.k.data_ptr(), x.v.data_ptr(), x.masks.data_ptr(), 3,
                                    4, 2, 64, 20, x.seq, 0, x.out.data_ptr(), x.ld, x.ws.data_ptr(), x.ws.numel(), None)
    assert bad() == -4
    rows = np.ones((5, 2, 64), np.float32)
    assert np.all(pkg.attn_decode(np.ones((4, 64), np.float32), rows, rows, 64, 0) == 1.0)
    y = Verify(3, 100, seed=15).setup(lib)
    st = stream()
    hip = C.CDLL("libamdhip64.so.7")
    x.out.fill_(NAN)
    torch.cuda.synchronize()
    assert hip.hipSetDevice(99) != 0  # leaves the runtime's last error set
    d = y.d
    rcs = [lib.tf_hip_attn_tree(0, F32, x.q.data_ptr(), x.ld, x.k.data_ptr(), x.v.data_ptr(), x.masks.data_ptr(), 3, 4, 2,
                                64, 20, x.seq, 0, x.out.data_ptr(), x.ld, x.ws.data_ptr(), x.ws.numel(), st),
           lib.tf_hip_verify_tree(0, d["logits"].data_ptr(), 100, 100, d["tokens"].data_ptr(), d["parent"].data_ptr(), 3,
                                  None, 0, 0.8, 1.0, d["draws"].data_ptr(), d["path"].data_ptr(), d["result"].data_ptr(),
                                  None, y.ws.data_ptr(), y.ws.numel(), st)]
    hip.hipGetLastError()
    assert rcs == [0, 0]
    torch.cuda.synchronize()
    assert torch.equal(x.out.view(3, 4, 64).double(), ok)
