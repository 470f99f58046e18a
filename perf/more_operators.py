"""Performance cases of the operators for several new tokens a sequence over paged caches.

A server that answers several conversations at once keeps their keys and values in pages
(`[pages][key_heads][page][dh]`, fp32 or fp16 values). Prompts come in together, of different
lengths, and where a small model drafts ahead, the tree of its tokens is checked in one step and
the path that the large model would have taken is kept. Kinds of case:

  prompt  every sequence's `new` tokens attend, each to the tokens up to its own: what the pages
          held before (`old`) and the new ones, causal (`paged_prompt`); the rows of all sequences
          one after another. `reach` and `gap`: a window's layers, and those that see what is behind it
  tree    the new tokens are drafted ones, a tree: each attends to the old tokens, its ancestors
          and itself (`paged_tree`)
  verify  the tree against the logits of its tokens: the path of the likeliest tokens through it,
          its length, and the token after it (`verify`)
  keep    a layer's keys and values of such a step: the drafted tokens' go into the pages
          (`paged_store`), and those of the path move together behind the old ones (`paged_keep`)

With `own` false the same is computed in elementary torch operations, sequences padded to the
longest.
"""

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
_DEV = "cuda" if torch.cuda.is_available() else "cpu"


def listed():
    attn = dict(ragged=True, heads=12, key_heads=4, dh=64, page=64, half=False)
    return [
        # the smallest model's first sentence: launches and host work count
        dict(attn, name="prompt-1x20", kind="prompt", n=1, new=20, old=0, ragged=False, heads=4, key_heads=2, dh=16,
             page=16, reach=0, gap=0),
        # one long document, fp32 pages
        dict(attn, name="prompt-1x8001", kind="prompt", n=1, new=8001, old=0, ragged=False, reach=0, gap=0),
        # a server's usual intake: prompts of many lengths over fp16 pages
        dict(attn, name="prompt-16x1500-half", kind="prompt", n=16, new=1500, old=0, half=True, reach=0, gap=0),
        # a chunk of each of six long conversations, in layers that see what their window has left
        dict(attn, name="prompt-6x256-far", kind="prompt", n=6, new=256, old=9000, reach=0, gap=4096),
        # second turns behind cached first ones in a window's layers, eight query heads on a key head of 128
        dict(attn, name="prompt-5x900-window", kind="prompt", n=5, new=900, old=3000, heads=16, key_heads=2, dh=128,
             page=32, half=True, reach=1024, gap=0),
        # one conversation's drafts behind a long cache
        dict(attn, name="tree-1x25", kind="tree", n=1, new=25, old=9001, ragged=False, reach=0, gap=0),
        # a batch with a large tree each over fp16 pages
        dict(attn, name="tree-24x48-half", kind="tree", n=24, new=48, old=6000, half=True, reach=0, gap=0),
        # many short conversations with few drafts, a key head a query head, small pages
        dict(attn, name="tree-40x7", kind="tree", n=40, new=7, old=900, heads=12, key_heads=12, page=16, reach=0, gap=0),
        # one tree's tokens looked over
        dict(name="verify-1x25", kind="verify", n=1, new=25, ragged=False, vocab=32000, half=False),
        # a batch's, fp16 mode's logits (equal ones among them)
        dict(name="verify-24x48", kind="verify", n=24, new=48, ragged=True, vocab=32000, half=True),
        # one conversation's drafts into a layer's pages, the path kept
        dict(attn, name="keep-1x25", kind="keep", n=1, new=25, old=1000, ragged=False),
        # a batch's, fp16 pages
        dict(attn, name="keep-64x48-half", kind="keep", n=64, new=48, old=600, heads=12, key_heads=12, half=True),
    ]


def _spread(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "tree", "tree", "verify", "keep"])
    half = rng.random() < 0.5
    if kind == "verify":
        n, new = _spread(rng, 1, 40), _spread(rng, 1, 64)
        most = min(150000, 30000000 // (n * new))
        return dict(kind=kind, n=n, new=new, ragged=rng.random() < 0.6,
                    vocab=rng.choice([min(32000, most), _spread(rng, 60, most), _spread(rng, 60, most)]), half=half)
    dh = rng.choice([64, 64, 64, 16, 32, 80, 128, 256])
    key_heads, group = rng.choice([(4, 3), (12, 1), (2, 8), (4, 2), (1, 16), (8, 1)])
    heads = key_heads * group
    case = dict(kind=kind, n=0, new=0, old=0, ragged=rng.random() < 0.7, heads=heads, key_heads=key_heads, dh=dh,
                page=rng.choice([16, 16, 32, 64, 64, 128, 256, 48]), half=half)
    slots = (200 << 20) // (8 * key_heads * dh)  # tokens that the pages may hold
    if kind == "prompt":
        # (the plain form holds every score, and the largest listed case's work is not passed)
        n = _spread(rng, 1, 24)
        new = _spread(rng, 2, 6000)
        room = min(slots // n, 400000000 // (n * heads * new), int(40e9 / (4 * heads * dh * n * new)))
        new = min(new, max(2, room // 2))
        old = rng.choice([0, 0, _spread(rng, 1, max(1, min(30000, room - new)))])
        return dict(case, n=n, new=new, old=old, reach=rng.choice([0, 0, 0, 1 + (new + old) // 4, 7]),
                    gap=rng.choice([0, 0, 0, (new + old) // 3]))
    n, new = _spread(rng, 1, 64), rng.randint(1, rng.choice([8, 64, 64, 200]))
    most = max(1, min(slots // n - new, 200000000 // (n * heads * new)))
    old = _spread(rng, 1, min(60000, most))
    case = dict(case, n=n, new=new, old=old)
    if kind == "tree":
        case.update(reach=rng.choice([0, 0, 0, 1 + old // 2]), gap=rng.choice([0, 0, 0, 3, old // 3]))
    return case


def _sizes(case):
    """The sequences' old and new tokens: all the most, or spread below it (the first's are the
    most), the same for every seed."""
    n, old, new = case["n"], case.get("old", 0), case["new"]
    if not case["ragged"]:
        return [old] * n, [new] * n
    u = [math.fmod(0.6180339887 * i, 1.0) for i in range(n)]
    w = [math.fmod(0.7548776662 * i, 1.0) for i in range(n)]
    return ([old if i == 0 else int(u[i] * (old + 1)) for i in range(n)],
            [new if i == 0 else 1 + int(w[i] * new) for i in range(n)])


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=_DEV)


def _layout(case, seed):
    """Lengths, the page table [n][width] (pages in no order, a tenth of them unused) and the
    number of pages."""
    old, new = _sizes(case)
    lens = np.array([a + b for a, b in zip(old, new)], np.int64)
    page = case["page"]
    used = -(-lens // page)
    total = int(used.sum())
    pages = total + total // 10 + 1
    ids = np.random.default_rng(seed).permutation(pages)[:total]
    table = np.zeros((len(lens), int(used.max())), np.int64)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = ids[at:at + u]
        at += u
    return lens, table, pages


def _trees(case, seed):
    """Each sequence's drafted tokens: [n][new] the node that each follows (-1: the old tokens; what
    is behind a sequence's last is -1 too), and the tokens. The first is the one picked last; the
    others hang below it, most of them near it."""
    rng = np.random.default_rng([seed, 1])
    _, new = _sizes(case)
    parent = np.full((case["n"], case["new"]), -1, np.int64)
    for b, f in enumerate(new):
        for i in range(1, f):
            parent[b, i] = int(rng.random() ** 1.5 * i)
    return parent, rng.integers(0, case.get("vocab", 32000), parent.shape).astype(np.int64)


def _ancestors(parent):
    """[n][new][new] whether node j is node i or one that it comes from, and [n][new] the nodes' depths."""
    n, f = parent.shape
    up = np.zeros((n, f, f), bool)
    for i in range(f):
        up[:, i, i] = True
        for b in range(n):
            if parent[b, i] >= 0:
                up[b, i] |= up[b, parent[b, i]]
    return up, up.sum(2) - 1


def _inputs(case, seed):
    """The tensors of a case, by name."""
    g = _generator(seed)
    n = case["n"]
    old, new = (np.array(x, np.int64) for x in _sizes(case))
    rows = int(new.sum())
    a = dict(old=old, new=new)
    if case["kind"] != "prompt":
        a["parent"], a["ids"] = _trees(case, seed)
    if case["kind"] == "verify":
        vocab = case["vocab"]
        x = _normal(g, rows, vocab) * 2.5
        # three drafted tokens of four are what the model would say
        parent, ids = a["parent"], a["ids"]
        first = np.cumsum(new) - new
        agree = np.random.default_rng([seed, 2]).random(parent.shape) < 0.75
        b, i = np.nonzero((parent >= 0) & agree)
        at = torch.from_numpy(first[b] + parent[b, i]).to(_DEV), torch.from_numpy(ids[b, i]).to(_DEV)
        x[at] = 16.0 + _normal(g, len(b))
        a["x"] = x.half().float() if case["half"] else x
        return a
    a["lens"], a["table"], a["pages"] = _layout(case, seed)
    KH, dh, page, H = case["key_heads"], case["dh"], case["page"], case["heads"]
    dtype = torch.float16 if case["half"] else torch.float32
    a["k"], a["v"] = (_normal(g, a["pages"], KH, page, dh).mul_(0.8).to(dtype) for _ in range(2))
    if case["kind"] == "keep":
        a["k_new"], a["v_new"] = (_normal(g, rows, KH, dh) * 0.8 for _ in range(2))
        # a path through each tree: from the first node, the eldest child of each, three times of four
        rng = np.random.default_rng([seed, 2])
        a["path"], a["count"] = np.full((n, case["new"]), -1, np.int64), np.ones(n, np.int64)
        for b in range(n):
            at, left = 0, [0]
            while rng.random() < 0.75 and (a["parent"][b, :new[b]] == at).any():
                at = int(np.argmax(a["parent"][b, :new[b]] == at))
                left.append(at)
            a["path"][b, :len(left)], a["count"][b] = left, len(left)
    else:
        a["q"] = _normal(g, rows, H, dh) * 1.8
    return a


def _rows(table, KH, page, L):
    """[n, KH, L]: the row of token t of a sequence's key head, over [pages][KH][page]."""
    t = torch.arange(L, device=table.device)
    pg = table[:, t // page]
    h = torch.arange(KH, device=table.device)
    return (pg[:, None] * KH + h[None, :, None]) * page + t % page


class _State:
    pass


# What one program keeps for its lifetime: a backend.
_BACKEND = []


def _package():
    """The package (its folder's name is not an identifier)."""
    if "slm_use_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location(
            "slm_use_amd", ROOT / "slm.use_amd" / "__init__.py",
            submodule_search_locations=[str(ROOT / "slm.use_amd")])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["slm_use_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["slm_use_amd"]


class _Buffers:
    """Device buffers of the backend, and torch's views of them; they go back with the last view."""

    def __init__(self, hip):
        self.hip, self.held = hip, []

    def like(self, shape, dtype=torch.float32, data=None):
        n = math.prod(shape)
        buf = self.hip.alloc_pages(*shape, half=True) if dtype == torch.float16 else self.hip.alloc(n)
        self.held.append(buf)
        kind = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4"}[dtype]
        view = torch.as_tensor(_View(self, buf, tuple(shape), kind), device="cuda")
        torch.cuda.synchronize()  # (the backend's stream has zeroed it)
        if data is not None:
            view.copy_(data)
        return buf, view

    def __del__(self):
        if self.hip.ctx:
            for b in self.held:
                b.free()


class _View:
    """A device buffer as torch takes it, holding its owner."""

    def __init__(self, owner, buf, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, data=(buf.ptr, False), version=2)


def _packed(case, new):
    """[rows] the place of each row of new tokens among sequences padded to `new`."""
    return np.nonzero((np.arange(case["new"]) < new[:, None]).ravel())[0]


def prepare(case, seed):
    s = _State()
    s.case, s.kind = case, case["kind"]
    a = _inputs(case, seed)
    n, F = case["n"], case["new"]
    if not own:
        a["at"] = _packed(case, a["new"])
        if s.kind in ("tree", "verify"):
            a["up"], a["depth"] = _ancestors(a["parent"])
        for name, v in a.items():
            setattr(s, name, torch.from_numpy(v).to(_DEV) if isinstance(v, np.ndarray) else v)
        return s
    # the backend's own buffers, and the sequences' handle
    pkg = _package()
    if not _BACKEND:
        _BACKEND.append(pkg.Hip(0))
    hip = s.hip = _BACKEND[0]
    mem = s.mem = _Buffers(hip)
    lens, page = a["old"] + a["new"], case.get("page", 64)
    table = a.get("table", np.zeros((n, 1 + int(lens.max()) // page), np.int64))
    s.seqs = hip.seqs(page, n, table.shape[1])
    s.seqs.set(lens, table, fresh=a["new"])
    if s.kind in ("tree", "verify"):
        there = np.arange(F) < a["new"][:, None]
        s.seqs.tree(a["parent"][there].astype(np.int32), a["ids"][there])
    rows = int(a["new"].sum())
    if s.kind == "verify":
        s.x, _ = mem.like(a["x"].shape, data=a["x"])
        s.count, count = mem.like((n,), torch.int32)
        s.path, path = mem.like((rows,), torch.int32)
        s.next, after = mem.like((n,), torch.int32)
        s.out = dict(count=count, path=path, next=after)
    else:
        KH, dh = case["key_heads"], case["dh"]
        dtype = a["k"].dtype
        s.k, k = mem.like(a["k"].shape, dtype, a["k"])
        s.v, v = mem.like(a["v"].shape, dtype, a["v"])
        s.cache = pkg.Pages(pages=a["pages"], page=page, key_heads=KH, dh=dh, k=s.k.ptr, v=s.v.ptr)
        if s.kind == "keep":
            s.k_new, _ = mem.like(a["k_new"].shape, data=a["k_new"])
            s.v_new, _ = mem.like(a["v_new"].shape, data=a["v_new"])
            s.count, _ = mem.like((n,), torch.int32, torch.from_numpy(a["count"]))
            s.path, _ = mem.like((rows,), torch.int32, torch.from_numpy(a["path"].ravel()[_packed(case, a["new"])]))
            s.out = dict(k=k, v=v)
        else:
            s.q, _ = mem.like(a["q"].shape, data=a["q"])
            s.y, y = mem.like(a["q"].shape)
            s.out = dict(y=y)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(s):
    c = s.case
    if not own:
        return {"prompt": _attend, "tree": _attend, "verify": _verify, "keep": _keep}[s.kind](s)
    if s.kind == "verify":
        s.hip.verify(s.seqs, s.count.ptr, s.path.ptr, s.next.ptr, s.x.ptr, c["vocab"])
    elif s.kind == "keep":
        s.hip.paged_store(s.seqs, s.cache, s.k_new.ptr, s.v_new.ptr)
        s.hip.paged_keep(s.seqs, s.cache, s.count.ptr, s.path.ptr)
    else:
        call = s.hip.paged_prompt if s.kind == "prompt" else s.hip.paged_tree
        call(s.seqs, s.cache, s.y.ptr, s.q.ptr, heads=c["heads"], scale=1.0 / math.sqrt(c["dh"]),
             reach=c["reach"] or None, gap=c["gap"])
    return s.out


def _attend(s):
    c = s.case
    n, F, H, KH, dh, page = c["n"], c["new"], c["heads"], c["key_heads"], c["dh"], c["page"]
    G = H // KH
    L = int(s.table.shape[1]) * page
    row = _rows(s.table, KH, page, L)
    keys, vals = s.k.view(-1, dh)[row].float(), s.v.view(-1, dh)[row].float()
    # rows of new tokens, sequences padded: [n, KH, F·G, dh]
    q = torch.zeros((n * F, H, dh), device=row.device)
    q[s.at] = s.q
    q = q.view(n, F, KH, G, dh).transpose(1, 2).reshape(n, KH, F * G, dh)
    t = torch.arange(L, device=row.device)
    i = torch.arange(F, device=row.device)
    old = s.old[:, None, None]
    if s.kind == "prompt":  # positions: a slot's number
        at, pos = t.expand(n, 1, L), s.old[:, None] + i
        line = (t < (s.old + s.new)[:, None])[:, None].expand(n, F, L)
    else:                   # a drafted token's is that of its depth
        j = (t - old).clamp(0, F - 1).expand(n, F, L)
        new = t >= old
        at = torch.where(new[:, 0], s.old[:, None] + s.depth.gather(1, j[:, 0]), t)[:, None]
        pos = s.old[:, None] + s.depth
        line = torch.where(new & (t < (s.old + s.new)[:, None, None]), s.up.gather(2, j), ~new)
    back = pos[:, :, None] - at
    sees = line & (back >= c["gap"])
    if c["reach"]:
        sees = sees & (back < c["reach"])
    sees = sees[:, None, :, None].expand(n, 1, F, G, L).reshape(n, 1, F * G, L)
    score = torch.matmul(q, keys.transpose(2, 3)) * (1.0 / math.sqrt(dh))
    score = torch.where(sees, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    y = torch.matmul(w, vals).view(n, KH, F, G, dh).transpose(1, 2).reshape(n * F, H, dh)
    return dict(y=y[s.at])


def _first_true(mask):
    """The lowest index that holds along the last axis, its length where none does."""
    at = torch.arange(mask.shape[-1], device=mask.device)
    return torch.where(mask, at, torch.full_like(at, mask.shape[-1])).amin(-1)


def _verify(s):
    n, F = s.parent.shape
    x = s.x
    picks = _first_true(x == x.amax(1, keepdim=True))
    pick = torch.full((n * F,), -1, dtype=torch.int64, device=x.device)
    pick[s.at] = picks
    pick = pick.view(n, F)
    i = torch.arange(F, device=x.device)
    there = i < s.new[:, None]
    # [n][node][child]: children that are what the model says behind the node, the eldest of them
    child = (s.parent[:, None, :] == i[:, None]) & (s.ids[:, None, :] == pick[:, :, None]) & there[:, None, :]
    eldest = _first_true(child)
    follows = (eldest.gather(1, s.parent.clamp(min=0)) == i) & (s.parent >= 0) | (i == 0)
    on = (follows[:, None, :] | ~s.up).all(2) & there  # a node all of whose line is
    count = on.sum(1)
    path = torch.sort(torch.where(on, i, torch.full_like(i, F)), dim=1)[0]
    last = path.gather(1, (count - 1)[:, None])
    path = torch.where(path < F, path, torch.full_like(path, -1)).view(-1)[s.at]
    return dict(count=count.to(torch.int32), path=path.to(torch.int32), next=pick.gather(1, last)[:, 0].to(torch.int32))


def _keep(s):
    c = s.case
    n, F, KH, dh, page = c["n"], c["new"], c["key_heads"], c["dh"], c["page"]
    L = int(s.table.shape[1]) * page
    row = _rows(s.table, KH, page, L)
    k, v = s.k.view(-1, dh), s.v.view(-1, dh)
    i = torch.arange(F, device=row.device)
    slot = (s.old[:, None] + i).clamp(max=L - 1)
    new = row.gather(2, slot[:, None].expand(n, KH, F)).transpose(1, 2).reshape(n * F, KH)[s.at].view(-1)
    k[new], v[new] = s.k_new.view(-1, dh).to(k.dtype), s.v_new.view(-1, dh).to(v.dtype)
    on = (i < s.count[:, None])[:, None].expand(n, KH, F)
    to = row.gather(2, slot[:, None].expand(n, KH, F))[on]
    frm = row.gather(2, (s.old[:, None] + s.path.clamp(min=0))[:, None].expand(n, KH, F))[on]
    k[to], v[to] = k[frm], v[frm]
    return dict(k=s.k, v=s.v)


# ---------------------------------------------------------------------------------------
# compulsory work
# ---------------------------------------------------------------------------------------

def work(case):
    c = case
    old, new = _sizes(c)
    rows = sum(new)
    if c["kind"] == "verify":
        return dict(bytes=4 * rows * c["vocab"] + 8 * c["n"] + 12 * rows, flops=rows * c["vocab"])
    KH, dh, unit = c["key_heads"], c["dh"], 2 if c["half"] else 4
    if c["kind"] == "keep":
        # the new rows, and what of the path moves (by the share that the inputs keep: about a path of three)
        return dict(bytes=2 * KH * dh * (rows * (4 + unit) + c["n"] * 4 * unit) + 8 * rows, flops=2 * rows * KH * dh)
    # pairs of a new token and one that it sees, and the tokens that some new token sees
    reach, gap = c["reach"] or 1 << 40, c["gap"]
    pairs = seen = 0
    if c["kind"] == "prompt":
        for o, f in zip(old, new):
            p = np.arange(o, o + f)
            pairs += int(np.maximum(0, np.maximum(0, p + 1 - gap) - np.maximum(0, p - reach + 1)).sum())
            seen += max(0, max(0, o + f - gap) - max(0, o - reach + 1))
    else:
        parent, _ = _trees(c, 0)
        up, depth = _ancestors(parent)
        for b, (o, f) in enumerate(zip(old, new)):
            p = o + depth[b, :f]
            pairs += int(np.maximum(0, np.minimum(o, np.maximum(0, p + 1 - gap)) - np.maximum(0, p - reach + 1)).sum())
            pairs += int(up[b, :f].sum()) if not gap else 0
            seen += max(0, min(o, max(0, int(p.max()) + 1 - gap)) - max(0, o - reach + 1)) + (f if not gap else 0)
    return dict(bytes=unit * 2 * KH * dh * seen + 8 * rows * c["heads"] * dh, flops=4 * c["heads"] * dh * pairs)


# ---------------------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    c, a = case, _inputs(case, seed)
    n = c["n"]
    first = np.cumsum(a["new"]) - a["new"]
    if c["kind"] == "verify":
        picks = np.argmax(a["x"].cpu().numpy(), axis=1)
        count, after = np.zeros(n, np.int32), np.zeros(n, np.int32)
        path = np.full(int(a["new"].sum()), -1, np.int32)
        for b in range(n):
            at, done = 0, 0
            while True:
                path[first[b] + done] = at
                done += 1
                said = picks[first[b] + at]
                then = [j for j in range(at + 1, a["new"][b]) if a["parent"][b, j] == at and a["ids"][b, j] == said]
                if not then:
                    break
                at = then[0]
            count[b], after[b] = done, said
        return dict(count=count, path=path, next=after)
    KH, dh, page = c["key_heads"], c["dh"], c["page"]
    k, v = a["k"].view(-1, dh), a["v"].view(-1, dh)

    def flat(b, h, t):
        pg = a["table"][b, t // page]
        return torch.from_numpy((pg * KH + h) * page + t % page).to(_DEV)

    if c["kind"] == "keep":
        for b in range(n):
            f = int(a["new"][b])
            for h in range(KH):
                at = flat(b, h, a["old"][b] + np.arange(f))
                kept = torch.from_numpy(a["path"][b, :a["count"][b]]).to(_DEV)
                for to, frm in ((k, a["k_new"]), (v, a["v_new"])):
                    new = frm[first[b]:first[b] + f, h].to(to.dtype)
                    to[at] = new
                    to[at[:len(kept)]] = new[kept]
        return dict(k=a["k"], v=a["v"])
    H, G = c["heads"], c["heads"] // KH
    reach, gap = c["reach"] or 1 << 40, c["gap"]
    if c["kind"] == "tree":
        up, depth = _ancestors(a["parent"])
    y = torch.zeros((int(a["new"].sum()), H, dh), dtype=torch.float64, device=_DEV)
    for b in range(n):
        o, f = int(a["old"][b]), int(a["new"][b])
        L = o + f
        for lo in range(0, f, 512):  # (rows of new tokens at a time)
            hi = min(f, lo + 512)
            pos = np.arange(L)
            if c["kind"] == "tree":
                pos[o:] = o + depth[b, :f]
            back = torch.from_numpy(pos[o + lo:o + hi]).to(_DEV)[:, None] - torch.from_numpy(pos).to(_DEV)
            sees = (back >= gap) & (back < reach)
            if c["kind"] == "tree":
                sees[:, o:] &= torch.from_numpy(up[b, lo:hi, :f]).to(_DEV)
            else:
                sees &= back >= 0
            none = ~sees.any(1)
            for h in range(KH):
                at = flat(b, h, np.arange(L))
                q = a["q"][first[b] + lo:first[b] + hi, h * G:(h + 1) * G].double()
                x = (q.reshape(-1, dh) @ k[at].double().T.contiguous()).view(hi - lo, G, L) / math.sqrt(dh)
                w = torch.softmax(x.masked_fill(~sees[:, None], -math.inf), -1).masked_fill(none[:, None, None], 0.0)
                y[first[b] + lo:first[b] + hi, h * G:(h + 1) * G] = (w.view(-1, L) @ v[at].double()).view(hi - lo, G, dh)
    return dict(y=y)
