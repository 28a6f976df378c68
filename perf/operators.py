"""Performance cases of the speculative-decoding operators: one step of a token loop that checks a
tree of drafted tokens against the model, at the shapes of the models that this repository's
benchmark and synthetic writer name (and one generic larger one).

A step drafts a tree of tokens (node 0 is the last token that is settled, a node's parent comes
before it), runs the model once over all nodes, and keeps the part of the tree that the model
agrees with. Of that step a case is one call:
  attn    one layer's attention of the tree's queries over the cache: every past position, and
          among the tree's own rows those that the node's mask names (tf_hip_attn_tree)
  verify  the walk down the tree by the target's probabilities, given draws and, where the drafts
          were sampled, the distributions they came from; the next token (tf_hip_verify_tree)
  keep    the accepted nodes' rows of every layer's cache moved up behind the settled ones
          (tf_hip_keep_path)

The plain forms are elementary torch operations: attention in float32, verification in float64
(its sums over a vocabulary and its comparisons with draws are next to a border).
"""
import math
import random

import numpy as np
import torch

DEV = "cuda"
F32, F16 = 0, 1  # cache types (ggml type codes)

own = False

# heads, kv heads, head size of one layer: Llama-3.2-1B, Qwen2.5-0.5B and Qwen2.5-1.5B shapes, and a
# larger generic one
HEADS = ((32, 8, 64), (14, 2, 64), (12, 2, 128), (64, 8, 128))
# layers, kv heads, head size of a whole cache, in the order of the first three
CACHES = ((16, 8, 64), (24, 2, 64), (28, 2, 128))
VOCABS = (32000, 128256, 151936)


def _attn(name, heads, n_tree, width, n_past, max_seq, layout, kv):
    h, g, hd = heads
    c = dict(kind="attn", heads=h, kv_heads=g, hd=hd, n_tree=n_tree, width=width, n_past=n_past, max_seq=max_seq,
             layout=layout, kv=kv)
    return dict(c, name=name) if name else c


def _verify(name, vocab, n_tree, width, sampled, temperature, top_p):
    # the parameters as the single-precision numbers that a sampler's are
    c = dict(kind="verify", vocab=vocab, n_tree=n_tree, width=width, sampled=sampled,
             temperature=float(np.float32(temperature)), top_p=float(np.float32(top_p)))
    return dict(c, name=name) if name else c


def _keep(name, cache, n_tree, n_path, n_past, max_seq, layout, kv):
    n_layer, g, hd = cache
    c = dict(kind="keep", layers=n_layer, kv_heads=g, hd=hd, n_tree=n_tree, n_path=n_path, n_past=n_past,
             max_seq=max_seq, layout=layout, kv=kv)
    return dict(c, name=name) if name else c


def listed():
    return [
        # The loop without a draft, right after a short question: one query over seven positions.
        _attn("attn_32x64_t1_past6", HEADS[0], 1, 1, 6, 512, 0, F32),
        # A chain of drafted tokens after a page of context, the usual n-gram or small-model draft.
        _attn("attn_32x64_t8_past1000", HEADS[0], 8, 1, 1000, 4096, 0, F32),
        # A ragged tree on the small model with seven query heads a kv head, head-major cache.
        _attn("attn_14x64_t37_past2029", HEADS[1], 37, 3, 2029, 4096, 1, F32),
        # A middling tree over the long-context workload's cache.
        _attn("attn_12x128_t26_past4096", HEADS[2], 26, 3, 4096, 8192, 1, F32),
        # A whole tree of 64 nodes over a long half-precision cache.
        _attn("attn_32x64_t64_past8191", HEADS[0], 64, 4, 8191, 16384, 0, F16),
        # The largest: many heads, a whole tree, a context of a book's chapter.
        _attn("attn_64x128_t64_past32768", HEADS[3], 64, 4, 32768, 40960, 0, F16),
        # Four drafted tokens in a chain, taken as the draft's likeliest; sampled at a temperature.
        _verify("verify_128k_t5_chain", 128256, 5, 1, False, 0.8, 1.0),
        # Drafts sampled from a small model, with its distributions at hand.
        _verify("verify_152k_t6_sampled", 151936, 6, 1, True, 0.7, 1.0),
        # A tree of likeliest tokens under a nucleus.
        _verify("verify_128k_t64_nucleus", 128256, 64, 4, False, 0.8, 0.95),
        # A tree of sampled tokens, several from one distribution, under a nucleus.
        _verify("verify_152k_t26_sampled_nucleus", 151936, 26, 3, True, 1.0, 0.9),
        # A short path out of a small tree on the 16-layer model; a longer one on the 28-layer model.
        _keep("keep_16x512_t16_path4", CACHES[0], 16, 4, 200, 512, 0, F32),
        _keep("keep_28x256_t64_path9", CACHES[2], 64, 9, 1501, 2048, 1, F32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "verify", "verify", "keep"))
    layout = rng.choice((0, 1))
    kv = rng.choice((F32, F16))
    if kind == "attn":
        heads = rng.choice(HEADS)
        n_tree = _log_int(rng, 1, 256)
        n_past = _log_int(rng, 1, 32768) - 1
        while n_tree * heads[0] * heads[2] * (n_past + n_tree) > 64 * 64 * 128 * 32768:
            n_tree = (n_tree + 1) // 2
        need = n_past + n_tree
        return _attn(None, heads, n_tree, rng.choice((1, 2, 3, 4)), n_past, need + rng.choice((0, 1, 100, 3001)), layout,
                     kv)
    if kind == "verify":
        return _verify(None, rng.choice(VOCABS) - rng.choice((0, 0, 1, 37)), _log_int(rng, 1, 64),
                       rng.choice((1, 2, 3, 4)), rng.choice((False, True)), rng.choice((0.0, 0.6, 0.8, 1.0)),
                       rng.choice((0.9, 0.95, 1.0)))
    n_tree = _log_int(rng, 2, 64)
    n_past = _log_int(rng, 1, 1900)
    return _keep(None, rng.choice(CACHES), n_tree, rng.randint(1, min(n_tree, 12)), n_past,
                 n_past + n_tree + rng.choice((0, 1, 77)), layout, kv)


# ---------------------------------------------------------------- inputs

def _tree(rng, n, width):
    """Parents of a tree of n nodes in which a node has at most `width` children: a chain for 1, else
    every node under a random earlier one with room."""
    parent, room = [-1], [width]
    for i in range(1, n):
        p = i - 1 if width == 1 else rng.choice([j for j in range(i) if room[j]])
        parent.append(p)
        room[p] -= 1
        room.append(width)
    return parent


def _ancestors(parent):
    """[n][n] truth values: node j is node i or above it."""
    n = len(parent)
    a = np.zeros((n, n), bool)
    for i, p in enumerate(parent):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def _mask_words(a):
    """Rows of truth values as 64-bit words, bit j % 64 of word j // 64 for column j."""
    n, m = a.shape
    w = (m + 63) // 64
    bits = np.zeros((n, w * 64), np.uint8)
    bits[:, :m] = a
    return np.packbits(bits, axis=1, bitorder="little").view(np.int64).copy()


def _cache_shape(c, layers=None):
    rows = (c["max_seq"], c["kv_heads"]) if c["layout"] == 0 else (c["kv_heads"], c["max_seq"])
    return (() if layers is None else (layers,)) + rows + (c["hd"],)


def prepare(case, seed):
    """The inputs of one call, on the GPU. The attention's caches hold no numbers behind the tree's rows, as
    memory that no token has been written to."""
    c, seed = case, int(seed)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = random.Random(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    s = dict(case)
    n = c["n_tree"]
    if c["kind"] == "attn":
        parent = _tree(rng, n, c["width"])
        s["masks"] = torch.from_numpy(_mask_words(_ancestors(parent))).to(DEV)
        # queries whose scores have a deviation near 2: a few positions hold most of a row's weight
        s["q"] = 2.0 * randn(n, c["heads"], c["hd"])
        t = torch.float32 if c["kv"] == F32 else torch.float16
        for name in ("k", "v"):
            x = randn(*_cache_shape(c))
            end = c["n_past"] + n
            (x[end:] if c["layout"] == 0 else x[:, end:]).fill_(float("nan"))
            s[name] = x.to(t)
        s["out"] = torch.empty_like(s["q"])
    elif c["kind"] == "verify":
        v = c["vocab"]
        parent = _tree(rng, n, c["width"])
        rank = [sum(parent[j] == parent[i] for j in range(i)) for i in range(n)]
        s["logits"] = 6.0 * randn(n, v)
        drafted = s["logits"] + randn(n, v)  # the draft model's idea of them
        at = torch.tensor([max(p, 0) for p in parent], device=DEV), torch.tensor(rank, device=DEV)
        if c["sampled"]:
            s["draft"] = torch.softmax(drafted / (c["temperature"] or 1.0), 1)
            some = torch.multinomial(s["draft"], max(rank) + 1, replacement=True, generator=gen)
        else:
            s["draft"] = None
            some = torch.topk(drafted, max(rank) + 1, 1).indices
        s["tokens"] = some[at].int()
        s["tokens"][0] = rng.randrange(v)
        s["parent"] = torch.tensor(parent, dtype=torch.int32, device=DEV)
        s["draws"] = torch.rand(n, generator=gen, device=DEV)
        s["path"] = torch.empty(n, dtype=torch.int32, device=DEV)
        s["result"] = torch.empty(2, dtype=torch.int32, device=DEV)
        s["probs"] = torch.empty(n, device=DEV)
    else:
        t = torch.float32 if c["kv"] == F32 else torch.float16
        for name in ("k", "v"):
            s[name] = randn(*_cache_shape(c, c["layers"])).to(t)
        path = [0] + sorted(rng.sample(range(1, n), c["n_path"] - 1)) if c["n_path"] > 1 else [0]
        s["path"] = torch.tensor(path + [-1] * (n - len(path)), dtype=torch.int32, device=DEV)
        s["result"] = torch.tensor([len(path), 0], dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------- the framework's calls

def _package():
    from __graft_entry__ import load_package
    return load_package()


def _workspace(s, nbytes):
    """The call's workspace, made once for a state as a program keeps one beside its cache."""
    if nbytes < 0:
        raise RuntimeError(f"workspace query failed with status {nbytes}")
    s["ws"] = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=DEV)
    return s["ws"]


def _own_attn(s):
    lib = _package().hip_lib()
    q, out = s["q"], s["out"]
    n, h, hd = q.shape
    ws = s.get("ws")
    if ws is None:
        ws = _workspace(s, lib.tf_hip_attn_tree_ws(n, h, s["kv_heads"], hd, s["n_past"]))
    rc = lib.tf_hip_attn_tree(q.device.index, s["kv"], q.data_ptr(), h * hd, s["k"].data_ptr(), s["v"].data_ptr(),
                              s["masks"].data_ptr(), n, h, s["kv_heads"], hd, s["n_past"], s["max_seq"], s["layout"],
                              out.data_ptr(), h * hd, ws.data_ptr(), ws.numel(),
                              torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError(f"tf_hip_attn_tree failed with status {rc}")
    return out


def _own_verify(s):
    lib = _package().hip_lib()
    logits, draft = s["logits"], s["draft"]
    n, v = logits.shape
    ws = s.get("ws")
    if ws is None:
        ws = _workspace(s, lib.tf_hip_verify_tree_ws(n, v))
    rc = lib.tf_hip_verify_tree(logits.device.index, logits.data_ptr(), v, v, s["tokens"].data_ptr(),
                                s["parent"].data_ptr(), n, None if draft is None else draft.data_ptr(), v,
                                s["temperature"], s["top_p"], s["draws"].data_ptr(), s["path"].data_ptr(),
                                s["result"].data_ptr(), s["probs"].data_ptr(), ws.data_ptr(), ws.numel(),
                                torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError(f"tf_hip_verify_tree failed with status {rc}")
    return {"path": s["path"], "result": s["result"], "probs": s["probs"]}


def _own_keep(s):
    lib = _package().hip_lib()
    rc = lib.tf_hip_keep_path(s["k"].device.index, s["kv"], s["k"].data_ptr(), s["v"].data_ptr(), s["layers"],
                              s["kv_heads"], s["hd"], s["n_past"], s["n_tree"], s["max_seq"], s["layout"],
                              s["path"].data_ptr(), s["result"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError(f"tf_hip_keep_path failed with status {rc}")
    return {"k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- the plain forms

def _plain_attn(s):
    n, h, hd = s["q"].shape
    g, past = s["kv_heads"], s["n_past"]
    end = past + n
    # [kv head][position][hd]
    k, v = (x[:end].permute(1, 0, 2) if s["layout"] == 0 else x[:, :end] for x in (s["k"], s["v"]))
    k, v = k.float().contiguous(), v.float().contiguous()
    q = s["q"].view(n, g, h // g, hd).permute(1, 0, 2, 3).reshape(g, n * (h // g), hd)
    score = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)
    j = torch.arange(n, device=DEV)
    see = (s["masks"][:, j // 64] >> (j % 64)) & 1 == 1
    see = torch.cat((torch.ones(n, past, dtype=torch.bool, device=DEV), see), 1)
    score = score.view(g, n, h // g, end).masked_fill(~see[None, :, None, :], -math.inf)
    top = score.amax(3, keepdim=True)
    p = torch.where(see[None, :, None, :], torch.exp(score - top), 0.0)
    p = p / p.sum(3, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.view(g, n * (h // g), end), v)
    return o.view(g, n, h // g, hd).permute(1, 0, 2, 3).reshape(n, h, hd)


def _plain_target(logits, temperature, top_p):
    """The distributions that tokens are sampled from, [n][vocab] in float64."""
    x = logits.double()
    if temperature <= 0:
        return torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
    p = torch.exp((x - x.amax(1, keepdim=True)) / temperature)
    p = p / p.sum(1, keepdim=True)
    if top_p < 1:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        sorted_p = p.gather(1, order)
        before = sorted_p.cumsum(1) - sorted_p
        kept = before < top_p
        kept[:, 0] = True
        p = p * torch.zeros_like(kept).scatter_(1, order, kept)
        p = p / p.sum(1, keepdim=True)
    return p


def _plain_verify(s):
    n = s["logits"].shape[0]
    p = _plain_target(s["logits"], s["temperature"], s["top_p"])
    up = s["parent"].long().clamp_min(0)
    tok, u = s["tokens"].long(), s["draws"].double()
    i = torch.arange(n, device=DEV)
    node = i > 0
    sibling = (s["parent"][:, None] == s["parent"][None, :]) & (i[None, :] < i[:, None]) & node[None, :]  # j before i
    rank = sibling.sum(1)
    kids = torch.zeros(n, dtype=torch.long, device=DEV).index_add_(0, up[1:], torch.ones_like(up[1:]))
    pc = p[up, tok]
    if s["draft"] is None:
        again = (sibling & (tok[:, None] == tok[None, :])).any(1)
        fresh = torch.where(again, 0.0, pc)
        before = (sibling * fresh[None, :]).sum(1)
        take = (fresh > 0) & (u * (1.0 - before) < fresh)
        left = p.clone()
        left[up[1:], tok[1:]] = 0.0
    else:
        q = s["draft"].double()
        qc = q[up, tok]
        t, mass = torch.zeros(n, 1, dtype=torch.float64, device=DEV), torch.ones(n, 1, dtype=torch.float64, device=DEV)
        take = torch.zeros(n, dtype=torch.bool, device=DEV)
        left = p
        for k in range(s["width"]):  # a node's k-th child against what its elder siblings' rejections leave
            rest = (pc - t[up, 0] * qc).clamp_min(0.0)
            take = take | ((rank == k) & (rest > 0) & (u * qc * mass[up, 0] < rest))
            t = torch.where((kids > k)[:, None], t + mass, t)
            left = (p - t * q).clamp_min(0.0)
            mass = left.sum(1, keepdim=True)
    take = (take & node) | ~node
    take = take & ~(sibling & take[None, :]).any(1)
    # a node is on the path where itself and all above it are taken
    above = (i[:, None] == i[None, :]) | (up[:, None] == i[None, :])
    for _ in range(n.bit_length()):
        above = torch.matmul(above.float(), above.float()) > 0
    on = ~(above & ~take[None, :]).any(1)
    count = on.sum()
    path = torch.where(i < count, torch.sort(torch.where(on, i, n)).values, -1)
    last = torch.where(on, i, -1).amax()
    w = left[last]
    w = torch.where(w.sum() > 0, w, p[last])
    total = w.cumsum(0)
    token = (total <= s["draws"][0].double() * total[-1]).sum()
    token = torch.minimum(token, torch.where(w > 0, torch.arange(w.numel(), device=DEV), 0).amax())
    probs = torch.where(node, pc, p[last, token]).float()
    return {"path": path.int(), "result": torch.stack((count, token)).int(), "probs": probs}


def _plain_keep(s):
    n, past = s["n_tree"], s["n_past"]
    count = s["result"][0]
    i = torch.arange(n, device=DEV)
    src = past + torch.where(i < count, s["path"].long(), i)  # rows behind the path stay
    for x in (s["k"], s["v"]):
        d = 1 if s["layout"] == 0 else 2
        x.narrow(d, past, n).copy_(x.index_select(d, src))
    return {"k": s["k"], "v": s["v"]}


def run(state):
    k = state["kind"]
    if own:
        return (_own_attn if k == "attn" else _own_verify if k == "verify" else _own_keep)(state)
    return (_plain_attn if k == "attn" else _plain_verify if k == "verify" else _plain_keep)(state)


# ---------------------------------------------------------------- work and exact results

def work(case):
    c = case
    n = c["n_tree"]
    if c["kind"] == "attn":
        h, hd, past = c["heads"], c["hd"], c["n_past"]
        size = 4 if c["kv"] == F32 else 2
        nbytes = 2 * (past + n) * c["kv_heads"] * hd * size + 2 * n * h * hd * 4 + n * ((n + 63) // 64) * 8
        return {"bytes": nbytes, "flops": 4 * n * h * hd * (past + (n + 1) / 2)}
    if c["kind"] == "verify":
        v = c["vocab"]
        return {"bytes": n * v * 4 * (2 if c["sampled"] else 1) + 24 * n, "flops": 4 * n * v}
    size = 4 if c["kv"] == F32 else 2
    return {"bytes": 2 * 2 * c["layers"] * c["n_path"] * c["kv_heads"] * c["hd"] * size, "flops": 0}


def _exact_attn(s):
    n, h, hd = s["q"].shape
    rep, past = h // s["kv_heads"], s["n_past"]
    words = s["masks"].cpu().numpy().view(np.uint64)
    see = np.ones((n, past + n), bool)
    see[:, past:] = [[(int(words[i, j // 64]) >> (j % 64)) & 1 for j in range(n)] for i in range(n)]
    hide = torch.from_numpy(~see).to(DEV)
    out = torch.zeros(n, h, hd, dtype=torch.float64, device=DEV)
    for g in range(s["kv_heads"]):
        k, v = ((x[: past + n, g] if s["layout"] == 0 else x[g, : past + n]).double() for x in (s["k"], s["v"]))
        for head in range(g * rep, (g + 1) * rep):
            a = (s["q"][:, head].double() @ k.t().contiguous()) * hd ** -0.5
            a[hide] = -math.inf
            out[:, head] = torch.softmax(a, 1) @ v
    return out


def _exact_verify(s):
    n, vocab = s["logits"].shape
    parent, tokens = s["parent"].tolist(), s["tokens"].tolist()
    draws = s["draws"].double().tolist()
    temperature, top_p = s["temperature"], s["top_p"]

    def target(i):
        x = s["logits"][i].cpu().numpy().astype(np.float64)
        if temperature <= 0:
            p = np.zeros(vocab)
            p[int(np.argmax(x))] = 1.0
            return p
        p = np.exp((x - x.max()) / temperature)
        p /= p.sum()
        if top_p < 1:
            order = np.argsort(-x, kind="stable")
            cut = int(np.searchsorted(np.cumsum(p[order]), top_p)) + 1  # up to the one that reaches top_p
            p[order[cut:]] = 0.0
            p /= p.sum()
        return p

    rows = [target(i) for i in range(n)]
    probs = np.array([0.0] + [rows[parent[i]][tokens[i]] for i in range(1, n)])
    path, at = [0], 0
    while True:
        r = rows[at].copy()
        q = None if s["draft"] is None else s["draft"][at].cpu().numpy().astype(np.float64)
        found = -1
        for c in (j for j in range(1, n) if parent[j] == at):
            x = tokens[c]
            have, ask = r[x], (1.0 if q is None else q[x])
            if have > 0 and draws[c] * ask < have:
                found = c
                break
            if q is None:
                r[x] = 0.0
            else:
                r = np.maximum(r - q, 0.0)
            if r.sum() > 0:
                r /= r.sum()
        if found < 0:
            break
        path.append(found)
        at = found
    w = r if r.sum() > 0 else rows[at]
    run_sum = np.cumsum(w)
    token = min(int(np.searchsorted(run_sum, draws[0] * run_sum[-1], side="right")), int(np.flatnonzero(w > 0)[-1]))
    probs[0] = rows[at][token]
    return {"path": np.array(path + [-1] * (n - len(path)), np.int32), "result": np.array([len(path), token], np.int32),
            "probs": probs}


def _exact_keep(s):
    done = {}
    path = s["path"].tolist()[: int(s["result"][0])]
    for name in ("k", "v"):
        x = s[name].double()
        rows = x if s["layout"] == 0 else x.transpose(1, 2)
        new = rows.clone()
        for i, node in enumerate(path):
            new[:, s["n_past"] + i] = rows[:, s["n_past"] + node]
        done[name] = new if s["layout"] == 0 else new.transpose(1, 2)
    return done


def exact(case, seed):
    s = prepare(case, seed)
    k = case["kind"]
    return (_exact_attn if k == "attn" else _exact_verify if k == "verify" else _exact_keep)(s)
