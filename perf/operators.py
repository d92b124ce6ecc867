"""The serving operators that are measured: a paged 8-bit key/value cache (append, read back), attention over it, and
sampling of the next token, over the sizes that an engine meets that serves one user or a batch of them.

Where `own` is false, `run` computes them in elementary torch operations; where it is true, through the library's C
ABI (sepia_amd.hip), a pass being one batch of it (begin, the ops, end) as an engine issues it. The state is the same
on both sides, in memory of the library's where `own` is true, since its calls take its own buffers.

The cache: a pool of pages of `page` tokens. Page p holds int8 codes, K as [kv head][token][dim] and then V as
[kv head][dim][token], and one f32 scale a (K or V, kv head): value = code * scale. A table gives each sequence's pages
in order.
"""
import math

import torch

# The library's buffers are handles over the tensors themselves (_Memory): both sides' state is made alike.
own = False

EPS = 1e-6


def listed():
    return [
        # decode for one user: the new token's keys (normed) and values of 8 layers
        dict(name="append_one", op="append", layers=8, seqs=1, new=1, ctx=20000, kv_heads=8, dim=128, page=16),
        # decode of an odd batch at ragged lengths: pages partly filled, scales that grow
        dict(name="append_batch", op="append", layers=4, seqs=61, new=1, ctx=8000, kv_heads=16, dim=128, page=32),
        # prompts: three of them, ragged, the cache's pages filled from the start or behind what is there
        dict(name="append_prompts", op="append", layers=1, seqs=3, new=2000, ctx=900, kv_heads=8, dim=128, page=16),
        # decode for one user over a long context: 4 layers of global attention with a relative-position band
        dict(name="decode_one", op="attn", layers=4, seqs=1, new=1, ctx=20001, heads=64, kv_heads=8, dim=128, page=16,
             window=0, rel=1024),
        # decode of a batch in sliding-window layers
        dict(name="decode_window", op="attn", layers=2, seqs=32, new=1, ctx=9000, heads=64, kv_heads=16, dim=128,
             page=16, window=512, rel=512),
        # decode of a ragged batch, from short contexts to long ones
        dict(name="decode_batch", op="attn", layers=1, seqs=48, new=1, ctx=12000, heads=64, kv_heads=8, dim=128,
             page=64, window=0, rel=1024),
        # several drafted tokens a sequence checked at once, narrow heads
        dict(name="decode_drafts", op="attn", layers=2, seqs=9, new=5, ctx=5000, heads=32, kv_heads=8, dim=64, page=32,
             window=0, rel=300),
        # a chunk of a prompt behind what is cached of it
        dict(name="prompt_chunk", op="attn", layers=1, seqs=1, new=500, ctx=1500, heads=64, kv_heads=8, dim=128,
             page=16, window=0, rel=1024),
        # whole prompts of several users, ragged, in a sliding-window layer
        dict(name="prompts_window", op="attn", layers=1, seqs=3, new=1400, ctx=700, heads=64, kv_heads=16, dim=128,
             page=64, window=512, rel=512),
        # the next token of one user, an odd vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=100003, pad=0, kind="mixed"),
        # the next tokens of a batch whose requests ask for different things
        dict(name="sample_batch", op="sample", rows=48, vocab=100003, pad=61, kind="mixed"),
        # nucleus sampling of a large batch over a large vocabulary, rows padded to whole lines
        dict(name="sample_nucleus", op="sample", rows=256, vocab=199999, pad=65, kind="nucleus"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "sample"])
    page, dim = rng.choice([16, 32, 64]), rng.choice([32, 64, 80, 128, 128, 128])
    if op == "append":
        seqs = _log(rng, 1, 64)
        return dict(op=op, layers=rng.randint(1, 4), seqs=seqs, new=_log(rng, 1, 3000 // seqs), ctx=_log(rng, 20, 8000),
                    kv_heads=rng.choice([1, 4, 8, 16]), dim=dim, page=page)
    if op == "attn":
        kv_heads, group = rng.choice([(8, 8), (16, 4), (4, 7), (2, 16), (8, 1), (3, 5)])
        new = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 600)])
        seqs = _log(rng, 1, 40 if new == 1 else max(1, min(12, 600 // new)))
        sliding = rng.random() < 0.5
        return dict(op=op, layers=rng.randint(1, 3) if new == 1 else 1, seqs=seqs, new=new,
                    ctx=_log(rng, 20, min(30000, 300000 // seqs) if new < 10 else 3000), heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, page=page, window=rng.choice([100, 512, 1024]) if sliding else 0,
                    rel=rng.choice([0, 300, 512, 1024]))
    return dict(op=op, rows=_log(rng, 1, 128), vocab=_log(rng, 1000, 200000), pad=rng.randint(0, 64),
                kind=rng.choice(["mixed", "nucleus", "top_k", "plain"]))


# ------------------------------------------------------------------- memory --
_device = None


def _dev():
    global _device
    if _device is None:
        from sepia_amd import hip
        _device = hip.Device()
    return _device


class _Memory:
    """A buffer of the library's over a tensor's own memory: nothing is copied or laid out beforehand. Given back with
    this object."""

    def __init__(self, t):
        dev = _dev()
        self.free, self.handle = dev.free, dev.wrap(t.data_ptr(), t.numel() * t.element_size())

    def __del__(self):
        if getattr(self, "handle", None):
            self.free(self.handle)


class Buf:
    """Device memory that holds `t`'s values: the tensor `t`, and in memory of the library's its `handle`."""

    def __init__(self, t):
        t = t.contiguous()
        if own:
            self.memory = _Memory(t)
            self.handle, self.t = self.memory.handle, t
        else:
            self.handle, self.t = None, t


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- sequences --
def _lengths(case):
    """Per sequence: tokens cached before the call, and new ones. The first has the case's lengths, the others are
    ragged below them; prompts (many new tokens) begin with nothing cached in every other sequence. They are the
    case's own, the same for every seed: outputs keep their shapes."""
    n, new, ctx = case["seqs"], case["new"], case["ctx"]
    g = torch.Generator().manual_seed(n * 7919 + new * 31 + ctx)
    r = torch.rand(n, 2, generator=g, dtype=torch.float64).tolist()
    have = [ctx if i == 0 else int(ctx * r[i][0] ** 1.5) for i in range(n)]
    add = [new if i == 0 or new < 10 else max(1, int(new * (0.3 + 0.7 * r[i][1]))) for i in range(n)]
    if new >= 10:
        have = [0 if i % 2 else h for i, h in enumerate(have)]
    return have, add


def _cache_inputs(case, seed, layer, have, add):
    """A pool with the sequences' pages in it, in a random order, a few pages free: codes of keys and values that were
    N(0, 1) and N(0, 0.5) (past each sequence's end too: what was there before), and the table."""
    g = _gen(seed, 1 + 10 * layer)
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    need = [-(-(h + a) // page) for h, a in zip(have, add)]
    pool = sum(need) + 5
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    codes = torch.empty(pool, 2, hk, page * d, dtype=torch.int8, device="cuda")
    scales = torch.empty(pool, 2, hk, dtype=torch.float32, device="cuda")
    for p0 in range(0, pool, 2048):
        x = _normal(g, min(pool, p0 + 2048) - p0, 2, hk, page * d) * torch.tensor([1.0, 0.5], device="cuda").view(2, 1, 1)
        s = x.abs().amax(-1) / 127
        scales[p0:p0 + 2048] = s
        codes[p0:p0 + 2048] = torch.round(x / s[..., None]).to(torch.int8)
    return codes.view(pool, -1), scales, table


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _inputs(case, seed, layer):
    """A layer's inputs by name, as torch tensors."""
    have, add = _lengths(case)
    codes, scales, table = _cache_inputs(case, seed, layer, have, add)
    starts = _starts(add)
    t, g = starts[-1], _gen(seed, 2 + 10 * layer)
    i = dict(codes=codes, scales=scales, table=table, lens=_int32(have), starts=_int32(starts))
    if case["op"] == "append":
        # the rows of every page that the call touches are read back
        first = [h // case["page"] * case["page"] for h in have]
        back = _starts([h + a - f for h, a, f in zip(have, add, first)])
        kv = case["kv_heads"] * case["dim"]
        i.update(k=_normal(g, t, kv, scale=2.0), v=_normal(g, t, kv, scale=0.5),
                 norm=1.0 + _normal(g, case["dim"], scale=0.1), first=_int32(first), back=_int32(back),
                 k_back=torch.zeros(back[-1], kv, device="cuda"), v_back=torch.zeros(back[-1], kv, device="cuda"))
        return i, have, add, starts, back
    pos = torch.cat([torch.arange(h, h + a) for h, a in zip(have, add)]).double()
    tau = torch.ones_like(pos) if case["window"] else 1.0 + 0.1 * torch.log((pos + 1) / 128.0).clamp(min=0.0)
    i.update(q=_normal(g, t, case["heads"], case["dim"]), tau=tau.float().cuda(),
             out=torch.zeros(t, case["heads"], case["dim"], device="cuda"))
    if case["rel"]:
        i["rel"] = _normal(g, t, case["heads"], case["rel"], scale=0.5)
    return i, have, add, starts, None


def _sample_inputs(case, seed):
    """Logits of a language model's kind (a few tokens far above a broad rest) and what each row asks for."""
    g = _gen(seed, 3)
    n, v = case["rows"], case["vocab"]
    x = _normal(g, n, v + case["pad"], scale=2.0)
    top = torch.randint(0, v, (n, 200), generator=g, device="cuda")
    x.scatter_add_(1, top, -2.5 * torch.log(torch.rand(n, 200, generator=g, device="cuda").clamp(min=1e-4)) + 3.0)
    r = torch.rand(n, 4, generator=g, device="cuda")
    temperature, top_p = 0.6 + 0.8 * r[:, 0], 0.5 + 0.49 * r[:, 1]
    min_p, top_k = 0.1 * r[:, 2], (1 + 100 * r[:, 3] ** 2).to(torch.int32)
    which = torch.arange(n, device="cuda") % 5   # mixed: nucleus, top-k and top-p, min-p, plain, greedy
    on = dict(mixed=(which < 2, which == 2, which == 1), nucleus=(which >= 0, which < 0, which < 0),
              top_k=(which < 0, which < 0, which >= 0), plain=(which < 0, which < 0, which < 0))[case["kind"]]
    if case["kind"] == "mixed":
        temperature = torch.where(which == 4, torch.zeros_like(temperature), temperature)
    return dict(logits=x, u=torch.rand(n, generator=g, device="cuda"), temperature=temperature,
                top_p=torch.where(on[0], top_p, torch.ones_like(top_p)),
                min_p=torch.where(on[1], min_p, torch.zeros_like(min_p)),
                top_k=torch.where(on[2], top_k, torch.zeros_like(top_k)),
                token=torch.zeros(n, dtype=torch.int32, device="cuda"), prob=torch.zeros(n, device="cuda"))


# ------------------------------------------------------------------ prepare --
def prepare(case, seed):
    state = {"case": dict(case), "layers": []}
    if case["op"] == "sample":
        state["layers"].append({k: Buf(t) for k, t in _sample_inputs(case, seed).items()})
    else:
        for layer in range(case["layers"]):
            i, have, add, starts, back = _inputs(case, seed, layer)
            state["layers"].append({k: Buf(t) for k, t in i.items()})
        # where each row of a call lies: its sequence and its place among the sequence's new rows
        seq = torch.cat([torch.full((a,), s) for s, a in enumerate(add)]).cuda()
        state["plan"] = dict(seq=seq, place=torch.arange(starts[-1], device="cuda") - _int32(starts)[seq].long(),
                             longest=max(h + a for h, a in zip(have, add)), most=max(add),
                             units=sum((h + a - 1) // case["page"] - h // case["page"] + 1 for h, a in zip(have, add)))
        if back:
            rows = [b - a for a, b in zip(back, back[1:])]
            seq = torch.cat([torch.full((a,), s) for s, a in enumerate(rows)]).cuda()
            state["plan"].update(back_seq=seq, back_place=torch.arange(back[-1], device="cuda") - _int32(back)[seq].long())
    if own:
        from sepia_amd import hip
        for b in state["layers"]:
            if case["op"] == "sample":
                state["desc"] = hip.SampleDesc(u=b["u"].handle, temperature=b["temperature"].handle,
                                               top_p=b["top_p"].handle, min_p=b["min_p"].handle,
                                               top_k=b["top_k"].handle)
            else:
                b["cache"] = hip.Kv8Cache(n_pages=b["scales"].t.shape[0], n_seqs=b["table"].t.shape[0],
                                          max_pages=b["table"].t.shape[1], n_kv_heads=case["kv_heads"],
                                          head_dim=case["dim"], page=case["page"], codes=b["codes"].handle,
                                          scales=b["scales"].handle, table=b["table"].handle)
    torch.cuda.synchronize()
    return state


# ---------------------------------------------------------------------- run --
def run(state):
    case = state["case"]
    if own:
        dev = _dev()
        dev.begin()
        for b in state["layers"]:
            _call(dev, case, state, b)
        dev.end()
    else:
        plain = dict(append=_plain_append, attn=_plain_attn, sample=_plain_sample)[case["op"]]
        for b in state["layers"]:
            plain(case, state.get("plan"), {k: x.t for k, x in b.items()})
    names = dict(append=("k_back", "v_back", "scales"), attn=("out",), sample=("token", "prob"))[case["op"]]
    return [{k: b[k].t for k in names} for b in state["layers"]]


def _call(dev, case, state, b):
    from ctypes import byref
    L, h = dev.L, {k: x.handle for k, x in b.items() if isinstance(x, Buf)}
    if case["op"] == "append":
        dev.check(L.sepia_hip_kv8_append(byref(b["cache"]), h["lens"], h["starts"], b["k"].t.shape[0], h["k"], h["v"],
                                         h["norm"], EPS), "kv8_append")
        dev.check(L.sepia_hip_kv8_read(byref(b["cache"]), h["first"], h["back"], b["k_back"].t.shape[0], h["k_back"],
                                       h["v_back"]), "kv8_read")
    elif case["op"] == "attn":
        dev.check(L.sepia_hip_kv8_attn(byref(b["cache"]), h["lens"], h["starts"], b["q"].t.shape[0], h["q"],
                                       h.get("rel"), h["tau"], h["out"], case["heads"], case["rel"], case["window"],
                                       1.0 / case["dim"]), "kv8_attn")
    else:
        dev.check(L.sepia_hip_sample(byref(state["desc"]), h["logits"], case["rows"], case["vocab"],
                                     case["vocab"] + case["pad"], h["token"], h["prob"]), "sample")


def _pages(case, codes):
    """The pool's codes as K [page][head][token][dim] and V [page][head][dim][token]."""
    p, hk, n, d = codes.shape[0], case["kv_heads"], case["page"], case["dim"]
    both = codes.view(p, 2, hk, n * d)
    return both[:, 0].view(p, hk, n, d), both[:, 1].view(p, hk, d, n)


def _plain_append(case, plan, b):
    """Values next to a rounding border decide a code, so they are computed in 64 bits."""
    page, hk, d, units = case["page"], case["kv_heads"], case["dim"], plan["units"]
    pos = b["lens"][plan["seq"]].long() + plan["place"]
    slot, at = pos % page, b["table"][plan["seq"], pos // page].long()
    head = (plan["place"] == 0) | (slot == 0)   # the first new row of a page
    unit = head.long().cumsum(0) - 1
    which = torch.zeros(units, dtype=torch.long, device="cuda").scatter_(0, unit, at)
    begin = torch.full((units,), page, dtype=torch.long, device="cuda").scatter_reduce_(0, unit, slot, "amin")
    k = b["k"].double().view(-1, hk, d)
    k = k * (1.0 / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS)) * b["norm"].double()
    kc, vc = _pages(case, b["codes"])
    for side, (x, codes) in enumerate(((k, kc), (b["v"].double().view(-1, hk, d), vc.transpose(2, 3)))):
        most = torch.zeros(units, hk, dtype=torch.float64, device="cuda")
        most.scatter_reduce_(0, unit[:, None].expand(-1, hk), x.abs().amax(-1), "amax")
        old = torch.where(begin[:, None] > 0, b["scales"][which, side], torch.zeros((), device="cuda"))
        scale = torch.maximum(old, (most.float() / 127))
        kept = torch.round(codes[which].double() * (old.double() / scale.double())[:, :, None, None])
        kept = torch.where(torch.arange(page, device="cuda")[:, None] < begin[:, None, None, None], kept,
                           codes[which].double())
        kept[unit, :, slot] = torch.round(x / scale[unit].double()[..., None]).clamp(-127, 127)
        codes[which] = kept.to(torch.int8)
        b["scales"][which, side] = scale
    pos = b["first"][plan["back_seq"]].long() + plan["back_place"]
    slot, at = pos % page, b["table"][plan["back_seq"], pos // page].long()
    b["k_back"].copy_((kc[at, :, slot].float() * b["scales"][at, 0][..., None]).flatten(1))
    b["v_back"].copy_((vc[at, :, :, slot].float() * b["scales"][at, 1][..., None]).flatten(1))


def _plain_attn(case, plan, b):
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    seqs, most, group = case["seqs"], plan["most"], case["heads"] // case["kv_heads"]
    first, pages = b["lens"].long() * 0, -(-plan["longest"] // page)
    if case["window"]:   # only the pages that a row of the sequence may see
        first = (b["lens"].long() - case["window"] + 1).clamp(min=0) // page
        pages = min(pages, (case["window"] + most) // page + 2)
    entry = (first[:, None] + torch.arange(pages, device="cuda")).clamp(max=b["table"].shape[1] - 1)
    at = b["table"].gather(1, entry).long()
    kc, vc = _pages(case, b["codes"])
    k = (kc[at].float() * b["scales"][at, 0][..., None, None]).permute(0, 2, 1, 3, 4).reshape(seqs * hk, -1, d)
    v = (vc[at].float() * b["scales"][at, 1][..., None, None]).permute(0, 2, 1, 4, 3).reshape(seqs * hk, -1, d)
    place = b["starts"][:-1].long()[:, None] + torch.arange(most, device="cuda")   # rows [seq][new], some past the last
    row = place.clamp(max=b["q"].shape[0] - 1)
    pos = b["lens"].long()[:, None] + torch.arange(most, device="cuda")
    q = b["q"][row].view(seqs, most, hk, group, d).permute(0, 2, 1, 3, 4).reshape(seqs * hk, most * group, d)
    s = torch.matmul(q, k.transpose(1, 2)).mul_(1.0 / d).view(seqs, hk, most, group, -1)
    dist = pos[:, :, None] - (first[:, None] * page + torch.arange(k.shape[1], device="cuda"))[:, None, :]
    if case["rel"]:
        rel = b["rel"][row].view(seqs, most, hk, group, -1).transpose(1, 2)
        near = dist.clamp(0, case["rel"] - 1)[:, None, :, None, :].expand(-1, hk, -1, group, -1)
        bias = rel.gather(4, near) * b["tau"][row][:, None, :, None, None]
        s += bias * (dist < case["rel"])[:, None, :, None, :]
    seen = (dist >= 0) & (dist < case["window"] if case["window"] else dist >= 0)
    s.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = (w / w.sum(-1, keepdim=True)).view(seqs * hk, most * group, -1)
    out = torch.matmul(w, v).view(seqs, hk, most, group, d).transpose(1, 2)
    b["out"].copy_(out[plan["seq"], plan["place"]].reshape(b["out"].shape))


def _plain_sample(case, plan, b):
    x, order = torch.sort(b["logits"][:, :case["vocab"]], dim=1, descending=True, stable=True)
    x = x.double()
    rank = torch.arange(case["vocab"], device="cuda")
    t = b["temperature"].double()[:, None]
    w = torch.where(t > 0, torch.exp((x - x[:, :1]) / t), (rank == 0).double())
    k = b["top_k"].long()[:, None]
    w = w * ((rank < k) | (k <= 0))
    below = w.cumsum(1) - w
    w = w * (below < b["top_p"].double()[:, None] * w.sum(1, keepdim=True)) * (w >= b["min_p"].double()[:, None])
    c = w.cumsum(1)
    last = (w > 0).sum(1) - 1
    pick = torch.minimum((c <= b["u"].double()[:, None] * c[:, -1:]).sum(1), last)[:, None]
    b["token"].copy_(order.gather(1, pick)[:, 0])
    b["prob"].copy_((w.gather(1, pick) / c[:, -1:])[:, 0])


# --------------------------------------------------------------------- work --
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 2 * n}
    have, add = _lengths(case)
    hk, d, n, layers = case["kv_heads"], case["dim"], sum(add), case["layers"]
    if case["op"] == "append":
        back = sum(h + a - h // case["page"] * case["page"] for h, a in zip(have, add))
        return {"bytes": layers * 2 * hk * d * (5 * n + 5 * back), "flops": layers * 2 * hk * d * 8 * n}
    seen = lambda p: min(p + 1, case["window"] or p + 1)  # noqa: E731
    cols = sum(seen(h + i) for h, a in zip(have, add) for i in range(a))
    rows = sum(h + a - max(0, h - (case["window"] or h + 1) + 1) for h, a in zip(have, add))
    band = sum(min(seen(h + i), case["rel"]) for h, a in zip(have, add) for i in range(a))
    kv = rows * 2 * hk * (d + 4 / case["page"])
    return {"bytes": layers * (kv + 4 * case["heads"] * (2 * n * d + band)), "flops": layers * 4 * d * case["heads"] * cols}


# -------------------------------------------------------------------- exact --
def exact(case, seed):
    if case["op"] == "sample":
        return [_exact_sample(case, _sample_inputs(case, seed))]
    one = _exact_append if case["op"] == "append" else _exact_attn
    return [one(case, *_inputs(case, seed, layer)) for layer in range(case["layers"])]


def _exact_append(case, i, have, add, starts, back):
    """Sequence by sequence, page by page: what the cache stands for after the call."""
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    k = i["k"].double().view(-1, hk, d)
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) / d + EPS) * i["norm"].double()
    new = (k, i["v"].double().view(-1, hk, d))
    scales, table = i["scales"].double().clone(), i["table"].tolist()
    read = ([], [])
    for s, (h, a) in enumerate(zip(have, add)):
        for p0 in range(h // page * page, h + a, page):
            at, lo, hi = table[s][p0 // page], max(h, p0), min(h + a, p0 + page)
            raw = i["codes"][at].view(2, hk, -1).double()
            held = (raw[0].view(hk, page, d).transpose(0, 1), raw[1].view(hk, d, page).permute(2, 0, 1))
            for side in (0, 1):
                x = new[side][starts[s] + lo - h:starts[s] + hi - h]
                scale = (x.abs().amax((0, 2)).float() / 127).double()
                c = torch.empty(0, hk, d, dtype=torch.float64, device="cuda")
                if lo > p0:
                    was = scales[at, side].clone()
                    scale = torch.maximum(scale, was)
                    c = torch.round(held[side][:lo - p0] * was[:, None] / scale[:, None])
                c = torch.cat([c, torch.round(x / scale[:, None]).clamp(-127, 127)])
                scales[at, side] = scale
                read[side].append(c * scale[:, None])
    return dict(k_back=torch.cat(read[0]).flatten(1), v_back=torch.cat(read[1]).flatten(1), scales=scales)


def _exact_attn(case, i, have, add, starts, back):
    page, hk, d, h_all = case["page"], case["kv_heads"], case["dim"], case["heads"]
    group, out = h_all // hk, []
    for s, (h, a) in enumerate(zip(have, add)):
        n = h + a
        pages = i["table"][s, :-(-n // page)].long()
        raw, scale = i["codes"][pages].view(-1, 2, hk, page * d).double(), i["scales"][pages].double()
        k = (raw[:, 0] * scale[:, 0, :, None]).view(-1, hk, page, d).transpose(1, 2).reshape(-1, hk, d)[:n]
        v = (raw[:, 1] * scale[:, 1, :, None]).view(-1, hk, d, page).permute(0, 3, 1, 2).reshape(-1, hk, d)[:n]
        rows = slice(starts[s], starts[s] + a)
        pos, col = torch.arange(h, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        dist = pos - col
        hidden = (dist < 0) | (dist >= (case["window"] or n + 1))
        y = torch.empty(a, h_all, d, dtype=torch.float64, device="cuda")
        for head in range(h_all):
            z = i["q"][rows, head].double() @ k[:, head // group].T.contiguous() / d
            if case["rel"]:
                b = i["rel"][rows, head].double().gather(1, dist.clamp(0, case["rel"] - 1)) * i["tau"][rows].double()[:, None]
                z = z + torch.where(dist < case["rel"], b, torch.zeros_like(b))
            z = z.masked_fill(hidden, -math.inf)
            e = torch.exp(z - z.max(1, keepdim=True).values)
            y[:, head] = e @ v[:, head // group].contiguous() / e.sum(1, keepdim=True)
        out.append(y)
    return dict(out=torch.cat(out))


def _exact_sample(case, i):
    import numpy as np
    x = i["logits"][:, :case["vocab"]].cpu().numpy().astype(np.float64)
    a = {k: i[k].cpu().numpy().astype(np.float64) for k in ("u", "temperature", "top_p", "min_p", "top_k")}
    token, prob = np.zeros(case["rows"], np.int32), np.zeros(case["rows"])
    for r in range(case["rows"]):
        order = np.argsort(-x[r], kind="stable")
        if a["temperature"][r] <= 0:
            token[r], prob[r] = order[0], 1.0
            continue
        if a["top_k"][r] > 0:
            order = order[:int(a["top_k"][r])]
        w = np.exp((x[r][order] - x[r][order[0]]) / a["temperature"][r])
        c = np.cumsum(w)
        n = 1 + int(np.sum(c[:-1] < a["top_p"][r] * c[-1]))
        n = max(1, min(n, int(np.sum(w >= a["min_p"][r]))))
        j = min(int(np.searchsorted(c[:n], a["u"][r] * c[n - 1], side="right")), n - 1)
        token[r], prob[r] = order[j], w[j] / c[n - 1]
    return dict(token=torch.from_numpy(token), prob=torch.from_numpy(prob))
