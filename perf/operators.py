"""Performance cases of the operators for several sequences over paged caches.

A server that answers several conversations at once keeps their keys and values in pages
(`[pages][key_heads][page][dh]`, fp32 or fp16 values) that it hands out as conversations grow,
and steps all of them together. Kinds of case:

  attend    one new token for each of n sequences: its key and value go into the pages
            (`paged_store`), then its query attends over the sequence's pages (`paged_attend`);
            with `mass`, the weight that every key received is added to what it had
  evict     every sequence of more than `keep` tokens gives up those whose keys received the
            least weight, the newest `recent` ones apart (`paged_evict`): what is kept behind
            the first `keep` slots moves into the slots that the evicted leave
  logprobs  m rows of logits: the log probability of a given token of each, the entropy, and
            the `top` likeliest tokens (`logprobs`)

With `own` false the same is computed in elementary torch operations.
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
    return [
        # the smallest model's first words: launches and host work count
        dict(name="attend-1x37", kind="attend", n=1, len=37, ragged=False, heads=4, key_heads=2, dh=16, page=16,
             half=False, mass=False, gap=0),
        # one long conversation of a model with global layers, which see what the window has left
        dict(name="attend-1x9001-far", kind="attend", n=1, len=9001, ragged=False, heads=12, key_heads=4, dh=64,
             page=64, half=False, mass=False, gap=4096),
        # a server's usual batch over fp16 pages, weights noted for an eviction
        dict(name="attend-24x6000-half", kind="attend", n=24, len=6000, ragged=True, heads=12, key_heads=4, dh=64,
             page=64, half=True, mass=True, gap=0),
        # many short conversations, a key head a query head, small pages
        dict(name="attend-64x2500", kind="attend", n=64, len=2500, ragged=True, heads=12, key_heads=12, dh=64,
             page=16, half=False, mass=False, gap=0),
        # two documents
        dict(name="attend-2x100003", kind="attend", n=2, len=100003, ragged=False, heads=12, key_heads=4, dh=64,
             page=256, half=False, mass=True, gap=0),
        # eight query heads on a key head of 128
        dict(name="attend-9x7777-wide", kind="attend", n=9, len=7777, ragged=True, heads=16, key_heads=2, dh=128,
             page=32, half=True, mass=True, gap=0),
        # a conversation that stays at its budget: sixteen tokens over it
        dict(name="evict-1x1040", kind="evict", n=1, len=1040, ragged=False, key_heads=4, dh=64, page=16, half=False,
             keep=1024, recent=64, steady=True),
        # a batch at its budget over fp16 pages, some of it below
        dict(name="evict-32x4200-half", kind="evict", n=32, len=4200, ragged=True, key_heads=4, dh=64, page=64,
             half=True, keep=4001, recent=256, steady=True),
        # long prompts that have just been read, cut to a quarter
        dict(name="evict-12x16384", kind="evict", n=12, len=16384, ragged=False, key_heads=12, dh=64, page=64,
             half=False, keep=4096, recent=512, steady=False),
        # a decode step's answer with its alternatives
        dict(name="logprobs-1x32000", kind="logprobs", m=1, n=32000, top=20, half=False, banned=0.0),
        # a prompt chunk's tokens scored, fp16 mode's logits (equal ones among them), some tokens forbidden
        dict(name="logprobs-256x32000", kind="logprobs", m=256, n=32000, top=5, half=True, banned=0.01),
        # a document scored over a larger vocabulary of odd size, no alternatives
        dict(name="logprobs-1021x65003", kind="logprobs", m=1021, n=65003, top=0, half=False, banned=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "evict", "logprobs"])
    half = rng.random() < 0.5
    if kind == "logprobs":
        n = rng.choice([97, 32000, _spread(rng, 50, 200000), _spread(rng, 50, 200000)])
        m = _spread(rng, 1, max(1, min(2000, 60000000 // n)))
        top = rng.choice([0, 1, 5, 20, rng.randint(2, 32)])
        if top and m * n > 20000000:  # (the plain form sorts the rows)
            top = 0
        return dict(kind=kind, m=m, n=n, top=min(top, n), half=half, banned=rng.choice([0.0, 0.0, 0.01, 0.3]))
    dh = rng.choice([64, 64, 64, 16, 32, 80, 128, 256])
    key_heads, group = rng.choice([(4, 3), (12, 1), (2, 8), (4, 2), (1, 16), (8, 1)])
    page = rng.choice([16, 16, 32, 64, 64, 128, 256, 48])
    most = (200 << 20) // (8 * key_heads * dh)  # tokens that the pages may hold
    if kind == "attend":
        n = _spread(rng, 1, 128)
        length = _spread(rng, 1, min(120000, max(1, most // n)))
        return dict(kind=kind, n=n, len=length, ragged=rng.random() < 0.7, heads=key_heads * group,
                    key_heads=key_heads, dh=dh, page=page, half=half, mass=rng.random() < 0.5,
                    gap=rng.choice([0, 0, 0, max(1, length // 3)]))
    n = _spread(rng, 1, 48)
    length = _spread(rng, 40, min(40000, max(40, most // n)))
    keep = rng.randint(max(1, length // 8), length)
    return dict(kind=kind, n=n, len=length, ragged=rng.random() < 0.6, key_heads=key_heads, dh=dh, page=page,
                half=half, keep=keep, recent=rng.randint(0, keep // 2), steady=rng.random() < 0.5)


def _lengths(case):
    """The sequences' lengths: all `len`, or spread below it (the first is `len`), the same for
    every seed; an evict case's lie around its budget."""
    n, top = case["n"], case["len"]
    if not case["ragged"]:
        return [top] * n
    u = [math.fmod(0.6180339887 * i, 1.0) for i in range(n)]
    if case["kind"] == "evict":
        low = max(1, case["keep"] - (top - case["keep"]))
        return [top if i == 0 else low + int(u[i] * (top - low)) for i in range(n)]
    return [top if i == 0 else 1 + int(u[i] * u[i] * (top - 1)) for i in range(n)]


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
    lens = np.array(_lengths(case), np.uint32)
    page = case["page"]
    used = -(-lens.astype(np.int64) // page)
    total = int(used.sum())
    pages = total + total // 10 + 1
    ids = np.random.default_rng(seed).permutation(pages)[:total].astype(np.uint32)
    table = np.zeros((len(lens), int(used.max())), np.uint32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = ids[at:at + u]
        at += u
    return lens, table, pages


def _inputs(case, seed):
    """The tensors of a case, by name."""
    g = _generator(seed)
    if case["kind"] == "logprobs":
        m, n = case["m"], case["n"]
        x = _normal(g, m, n) * 2.5
        # a few tokens stand out, as in a model's logits
        far = torch.randint(n, (m, min(n, 8)), generator=g, device=_DEV)
        x.scatter_add_(1, far, 3.0 + 2.0 * _normal(g, *far.shape))
        ids = torch.where(torch.rand(m, generator=g, device=_DEV) < 0.5, x.argmax(1),
                          torch.randint(n, (m,), generator=g, device=_DEV))
        if case["banned"]:
            x.masked_fill_(torch.rand((m, n), generator=g, device=_DEV) < case["banned"], -math.inf)
        if case["half"]:
            x = x.half().float()
        return dict(x=x, ids=ids)
    lens, table, pages = _layout(case, seed)
    KH, dh, page, n = case["key_heads"], case["dh"], case["page"], case["n"]
    dtype = torch.float16 if case["half"] else torch.float32
    a = dict(lens=lens, table=table, pages=pages)
    a["k"], a["v"] = (_normal(g, pages, KH, page, dh).mul_(0.8).to(dtype) for _ in range(2))
    if case["kind"] == "attend":
        a["q"] = _normal(g, n, case["heads"], dh) * 1.8
        a["k_new"], a["v_new"] = (_normal(g, n, KH, dh) * 0.8 for _ in range(2))
        a["seen"] = lens
        if case["mass"]:
            a["mass"] = torch.rand((pages, KH, page), generator=g, device=_DEV) * 3.0
        return a
    # what the keys have received so far: a few of them most of it, some nothing
    mass = torch.exp(2.0 * _normal(g, pages, KH, page) - 4.0)
    a["mass"] = torch.where(torch.rand(mass.shape, generator=g, device=_DEV) < 0.02, torch.zeros_like(mass), mass)
    # positions: in order of the slots after a prompt; after earlier evictions the first `keep`
    # slots hold what was kept, in no order, and the newest come behind
    L, keep = int(lens.max()), case["keep"]
    t = torch.arange(L, device=_DEV)
    born = t.expand(n, KH, L).clone()
    seen = lens.copy()
    if case["steady"]:
        old = min(keep, L)
        born[..., :old] = torch.argsort(torch.rand((n, KH, 2 * old), generator=g, device=_DEV), -1)[..., :old]
        born[..., old:] += old
        seen = (lens + old).astype(np.uint32)
        # (a sequence below the budget: nothing newer than its length)
        short = torch.from_numpy(lens.astype(np.int64)).to(_DEV) < old
        born[short] = t.expand(KH, L)
        seen = np.where(lens < old, lens, seen).astype(np.uint32)
    lens_d = torch.from_numpy(lens.astype(np.int64)).to(_DEV)
    row = _rows(torch.from_numpy(table.astype(np.int64)).to(_DEV), KH, page, L)
    valid = (t < lens_d[:, None, None]).expand(n, KH, L)
    a["born"] = torch.zeros((pages, KH, page), dtype=torch.int32, device=_DEV)
    a["born"].view(-1)[row[valid]] = born[valid].to(torch.int32)
    a["seen"] = seen
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


def prepare(case, seed):
    s = _State()
    s.case, s.kind = case, case["kind"]
    a = _inputs(case, seed)
    if not own:
        for name, v in a.items():
            if isinstance(v, np.ndarray):
                v = torch.from_numpy(v.astype(np.int64)).to(_DEV)
            setattr(s, name, v)
        if s.kind != "logprobs":  # what a call writes for part of the slots alone
            shape = (s.pages, case["key_heads"], case["page"])
            s.mass_out = torch.zeros(shape, device=_DEV)
            s.born_out = torch.zeros(shape, dtype=torch.int32, device=_DEV)
        return s
    # the backend's own buffers, and the sequences' handle
    pkg = _package()
    if not _BACKEND:
        _BACKEND.append(pkg.Hip(0))
    hip = s.hip = _BACKEND[0]
    mem = s.mem = _Buffers(hip)
    if s.kind == "logprobs":
        m, top = case["m"], case["top"]
        s.x, _ = mem.like(a["x"].shape, data=a["x"])
        s.ids = a["ids"].cpu().numpy().astype(np.uint32)
        s.lp, lp = mem.like((m,))
        s.ent, ent = mem.like((m,))
        s.out = dict(lp=lp, entropy=ent)
        s.top_ids = s.top_lp = None
        if top:
            s.top_ids, s.out["top_ids"] = mem.like((m, top), torch.int32)
            s.top_lp, s.out["top_lp"] = mem.like((m, top))
    else:
        KH, page, dh, n = case["key_heads"], case["page"], case["dh"], case["n"]
        pages, dtype = a["pages"], a["k"].dtype
        s.k, k = mem.like(a["k"].shape, dtype, a["k"])
        s.v, v = mem.like(a["v"].shape, dtype, a["v"])
        s.out = dict(k=k, v=v)
        s.seqs = hip.seqs(page, n, a["table"].shape[1])
        s.seqs.set(a["lens"], a["table"], seen=a["seen"])
        s.cache = pkg.Pages(pages=pages, page=page, key_heads=KH, dh=dh, k=s.k.ptr, v=s.v.ptr)
        shape = (pages, KH, page)
        s.mass_out = s.born_out = None
        if "mass" in a:
            s.mass, _ = mem.like(shape, data=a["mass"])
            s.mass_out, s.out["mass"] = mem.like(shape)
            s.cache.mass = s.mass.ptr
        if s.kind == "attend":
            s.q, _ = mem.like(a["q"].shape, data=a["q"])
            s.k_new, _ = mem.like(a["k_new"].shape, data=a["k_new"])
            s.v_new, _ = mem.like(a["v_new"].shape, data=a["v_new"])
            s.y, s.out["y"] = mem.like(a["q"].shape)
        else:
            s.born, _ = mem.like(shape, torch.int32, a["born"])
            s.born_out, s.out["born"] = mem.like(shape, torch.int32)
            s.cache.born = s.born.ptr
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(s):
    c = s.case
    if not own:
        return {"attend": _attend, "evict": _evict, "logprobs": _logprobs}[s.kind](s)
    if s.kind == "attend":
        s.hip.paged_store(s.seqs, s.cache, s.k_new.ptr, s.v_new.ptr)
        s.hip.paged_attend(s.seqs, s.cache, s.y.ptr, s.q.ptr, heads=c["heads"], gap=c["gap"],
                           scale=1.0 / math.sqrt(c["dh"]), mass_out=s.mass_out.ptr if s.mass_out else None)
    elif s.kind == "evict":
        s.hip.paged_evict(s.seqs, s.cache, s.mass_out.ptr, s.born_out.ptr, keep=c["keep"], recent=c["recent"])
    else:
        s.hip.logprobs(s.lp.ptr, s.x.ptr, s.ids, c["n"], entropy=s.ent.ptr, top=c["top"],
                       top_ids=s.top_ids.ptr if s.top_ids else None, top_lp=s.top_lp.ptr if s.top_lp else None)
    return s.out


def _attend(s):
    c = s.case
    n, H, KH, dh, page = c["n"], c["heads"], c["key_heads"], c["dh"], c["page"]
    L = s.table.shape[1] * page
    row = _rows(s.table, KH, page, L)
    k, v = s.k.view(-1, dh), s.v.view(-1, dh)
    new = row.gather(2, (s.lens - 1)[:, None, None].expand(n, KH, 1)).view(-1)
    k[new] = s.k_new.view(-1, dh).to(k.dtype)
    v[new] = s.v_new.view(-1, dh).to(v.dtype)
    sees = torch.arange(L, device=row.device) < (s.lens - c["gap"])[:, None]
    keys, vals = k[row].float(), v[row].float()
    q = s.q.view(n, KH, H // KH, dh)
    score = torch.matmul(q, keys.transpose(2, 3)) * (1.0 / math.sqrt(dh))
    score = torch.where(sees[:, None, None], score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    out = dict(k=s.k, v=s.v, y=torch.matmul(w, vals).view(n, H, dh))
    if c["mass"]:
        s.mass.view(-1)[new] = 0.0
        there = (torch.arange(L, device=row.device) < s.lens[:, None])[:, None].expand(n, KH, L)
        at = row[there]
        s.mass_out.view(-1)[at] = s.mass.view(-1)[at] + w.sum(2)[there]
        out["mass"] = s.mass_out
    return out


def _evict(s):
    c = s.case
    n, KH, dh, page, keep = c["n"], c["key_heads"], c["dh"], c["page"], c["keep"]
    L = s.table.shape[1] * page
    row = _rows(s.table, KH, page, L)
    t = torch.arange(L, device=row.device)
    there = (t < s.lens[:, None])[:, None].expand(n, KH, L)
    mass, born = s.mass.view(-1)[row], s.born.view(-1)[row].long()
    newest = there & (born + c["recent"] >= s.seen[:, None, None])
    key = torch.where(newest, torch.full_like(mass, math.inf), mass)
    key = torch.where(there, key, torch.full_like(mass, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(2, order, t.expand(n, KH, L))
    kept = there & (rank < keep)
    to, frm = row[there & ~kept & (t < keep)], row[kept & (t >= keep)]
    stay = row[kept & (t < keep)]
    k, v = s.k.view(-1, dh), s.v.view(-1, dh)
    k[to], v[to] = k[frm], v[frm]
    for new, old in ((s.mass_out, s.mass), (s.born_out, s.born)):
        new.view(-1)[stay] = old.view(-1)[stay]
        new.view(-1)[to] = old.view(-1)[frm]
    return dict(k=s.k, v=s.v, mass=s.mass_out, born=s.born_out)


def _logprobs(s):
    top = s.x.amax(1, keepdim=True)
    x = s.x - top
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    ex = torch.where(e > 0, e * x, torch.zeros_like(e))
    out = dict(lp=(x.gather(1, s.ids[:, None]) - log_total)[:, 0],
               entropy=(log_total - ex.sum(1, keepdim=True) / total)[:, 0])
    k = s.case["top"]
    if k:
        val, at = torch.sort(x, dim=1, descending=True, stable=True)
        out["top_ids"] = at[:, :k].to(torch.int32)
        out["top_lp"] = val[:, :k] - log_total
    return out


# ---------------------------------------------------------------------------------------
# compulsory work
# ---------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "logprobs":
        m, n = c["m"], c["n"]
        return dict(bytes=4 * m * n + m * (12 + 8 * c["top"]), flops=6 * m * n)
    lens = _lengths(c)
    KH, dh, unit = c["key_heads"], c["dh"], 2 if c["half"] else 4
    if c["kind"] == "attend":
        seen = sum(max(0, x - c["gap"]) for x in lens)
        nbytes = unit * 2 * KH * dh * (seen + c["n"]) + 8 * c["n"] * (c["heads"] + KH) * dh
        if c["mass"]:
            nbytes += 8 * KH * sum(lens)
        return dict(bytes=nbytes, flops=4 * c["heads"] * dh * seen)
    # the weights and positions of all, those of the kept; keys and values that move (a kept one
    # is behind the budget as often as not where none is newer: by the share of slots there)
    nbytes = 0
    for x in lens:
        kept = min(x, c["keep"])
        nbytes += 8 * KH * (x + kept)
        if x > c["keep"]:
            behind = min(x - c["keep"], c["recent"])
            behind += (kept - c["recent"]) * (x - c["keep"] - behind) // max(1, x - c["recent"])
            nbytes += 4 * unit * KH * dh * behind
    return dict(bytes=nbytes, flops=2 * KH * sum(lens))


# ---------------------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------------------

def _flat(a, b, h, KH, page, length):
    """The flat rows of sequence b's first `length` tokens under key head h."""
    t = np.arange(length)
    return torch.from_numpy((a["table"][b, t // page].astype(np.int64) * KH + h) * page + t % page).to(_DEV)


def exact(case, seed):
    c, a = case, _inputs(case, seed)
    if c["kind"] == "logprobs":
        m, k = c["m"], c["top"]
        out = dict(lp=[], entropy=[], **(dict(top_ids=[], top_lp=[]) if k else {}))
        for lo in range(0, m, 64):
            x = a["x"][lo:lo + 64].double()
            lse = torch.logsumexp(x, 1, keepdim=True)
            l = x - lse
            out["lp"].append(l.gather(1, a["ids"][lo:lo + 64, None])[:, 0])
            out["entropy"].append(-torch.where(torch.isinf(l), torch.zeros_like(l), l.exp() * l).sum(1))
            if k:
                at = np.argsort(-a["x"][lo:lo + 64].cpu().numpy(), axis=1, kind="stable")[:, :k]
                out["top_ids"].append(torch.from_numpy(at.astype(np.int32)))
                out["top_lp"].append(l.cpu().gather(1, torch.from_numpy(at)))
        return {name: torch.cat(v) for name, v in out.items()}
    KH, dh, page, n = c["key_heads"], c["dh"], c["page"], c["n"]
    k, v = a["k"].view(-1, dh), a["v"].view(-1, dh)
    if c["kind"] == "attend":
        H, G = c["heads"], c["heads"] // KH
        y = torch.zeros((n, H, dh), dtype=torch.float64, device=_DEV)
        mass = torch.zeros(a["pages"] * KH * page, dtype=torch.float64, device=_DEV)
        for b in range(n):
            length = int(a["lens"][b])
            sees = max(0, length - c["gap"])
            for h in range(KH):
                at = _flat(a, b, h, KH, page, length)
                k[at[-1]], v[at[-1]] = a["k_new"][b, h].to(k.dtype), a["v_new"][b, h].to(v.dtype)
                if c["mass"]:
                    a["mass"].view(-1)[at[-1]] = 0.0
                    mass[at] = a["mass"].view(-1)[at].double()
                if sees:
                    qs = a["q"][b, h * G:(h + 1) * G].double()
                    w = torch.softmax((k[at[:sees]].double() @ qs.T).T / math.sqrt(dh), -1)
                    y[b, h * G:(h + 1) * G] = w @ v[at[:sees]].double()
                    if c["mass"]:
                        mass[at[:sees]] += w.sum(0)
        out = dict(k=a["k"], v=a["v"], y=y)
        if c["mass"]:
            out["mass"] = mass.view(a["pages"], KH, page)
        return out
    mass, born = a["mass"].view(-1), a["born"].view(-1)
    mass_out, born_out = torch.zeros_like(mass, dtype=torch.float64), torch.zeros_like(born)
    for b in range(n):
        length = int(a["lens"][b])
        left = min(length, c["keep"])
        for h in range(KH):
            at = _flat(a, b, h, KH, page, length)
            w, p = mass[at].cpu().numpy(), born[at].cpu().numpy().astype(np.int64)
            newest = p >= int(a["seen"][b]) - c["recent"]
            keep = np.sort(np.lexsort((np.arange(length), -w, ~newest))[:left])
            gone = np.setdiff1d(np.arange(left), keep)
            frm = np.arange(left)
            frm[gone] = keep[keep >= left]
            frm = torch.from_numpy(frm).to(_DEV)
            k[at[:left]], v[at[:left]] = k[at[frm]], v[at[frm]]
            mass_out[at[:left]], born_out[at[:left]] = mass[at[frm]].double(), born[at[frm]]
    shape = (a["pages"], KH, page)
    return dict(k=a["k"], v=a["v"], mass=mass_out.view(shape), born=born_out.view(shape))
