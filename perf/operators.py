"""Measured cases of the batched-generation operators: rotary positions, appending keys and values to a paged
cache with the rotation applied on the way, attention over a prefix that the whole batch shares, and
verification of drafted tokens.

`run` computes an operator in its plain form (elementary torch operations, 32 bits, 64 where a far
position's angle or a long sum needs them), or, where `own` is true, by the framework's calls.

Shapes shared by the last three operators: the batch's new tokens are packed, sequence b has rows
start[b] .. start[b + 1] - 1 of them, len[b] tokens of its own in the cache (the new ones included), and a row
of page numbers; every sequence stands behind the same prefix of `prefix` tokens, whose pages `prefix_pages` lists.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"fp32": 0, "bf16": 1, "fp16": 2}
SCALINGS = {"none": 0, "linear": 1, "base": 2, "parts": 3}


# ------------------------------------------------------------------------------------------------ cases
def _rope(name, rows, heads, dim, rot, layout, scaling, dtype, far, inverse, packed):
    return {"name": name, "op": "rope", "rows": rows, "heads": heads, "dim": dim, "rot": rot, "layout": layout,
            "scaling": scaling, "dtype": dtype, "far": far, "inverse": inverse, "packed": packed}


def _append(name, batch, low, new, q_heads, kv_heads, dim, rot, layout, src, dtype, page, prefix, longest, packed, ragged):
    return {"name": name, "op": "append", "batch": batch, "low": low, "new": new, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "rot": rot, "layout": layout, "src": src, "dtype": dtype, "page": page,
            "prefix": prefix, "longest": longest, "packed": packed, "ragged": ragged}


def _attend(name, batch, low, new, q_heads, kv_heads, dim, dtype, page, prefix, longest, ragged):
    return {"name": name, "op": "attend", "batch": batch, "low": low, "new": new, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "prefix": prefix, "longest": longest,
            "ragged": ragged}


def _verify(name, batch, new, vocab, pad, ragged):
    return {"name": name, "op": "verify", "batch": batch, "new": new, "vocab": vocab, "pad": pad, "ragged": ragged}


def listed():
    return [
        # the character language model's queries in training: 64 sequences of 128 tokens, 4 heads of 32, fp32
        _rope("rope_char_lm_fp32", 8192, 4, 32, 32, "half", "none", "fp32", 128, False, False),
        # the gradient of a long-context step: half of each head rotated, scaled by parts, far positions
        _rope("rope_long_bf16_grad", 16384, 40, 128, 64, "interleaved", "parts", "bf16", 131072, True, True),
        # one user, one token, the character model's heads: latency
        _append("append_one_token", 1, 1, 1, 4, 4, 32, 32, "half", "fp32", "bf16", 16, 0, 97, False, 1),
        # a generation step with up to four drafted tokens a user, from one packed projection
        _append("append_drafts", 64, 1, 5, 32, 8, 128, 128, "half", "bf16", "bf16", 64, 2029, 700, True, 2),
        # prompts of several users in one pass, odd lengths
        _append("append_prompts", 7, 300, 2048, 32, 8, 128, 96, "interleaved", "fp16", "fp16", 32, 512, 2100, False, 3),
        # the character model's shape: 4 heads of 32, its 128 positions split between a prompt that all share and replies
        _attend("attend_char_lm", 16, 1, 1, 4, 4, 32, "bf16", 16, 96, 32, 4),
        # a chat step: one token a user behind a shared system prompt
        _attend("attend_chat", 32, 1, 1, 32, 8, 128, "bf16", 64, 2029, 700, 5),
        # drafted tokens under verification, eight query heads to a key head, pages of 16
        _attend("attend_drafts", 64, 1, 5, 32, 4, 64, "fp16", 16, 4001, 513, 6),
        # many users, long shared documents, long replies
        _attend("attend_large", 128, 2, 5, 32, 8, 128, "bf16", 64, 16384, 2048, 7),
        # the character model's 65 characters
        _verify("verify_char_lm", 64, 5, 65, 0, 8),
        # one user, a large vocabulary: latency
        _verify("verify_one", 1, 8, 131072, 0, 9),
        # many users, odd vocabulary in padded rows
        _verify("verify_batch", 192, 6, 100003, 93, 10),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rope", "append", "attend", "verify"))
    ragged = rng.randrange(1 << 20)
    if op == "rope":
        dim = rng.choice((32, 64, 96, 128, 256))
        heads = _log(rng, 1, 64)
        rows = _log(rng, 1, min(32768, 80_000_000 // (heads * dim)))
        c = _rope("", rows, heads, dim, rng.choice((dim, dim // 2, dim - 8)), rng.choice(("half", "interleaved")),
                  rng.choice(tuple(SCALINGS)), rng.choice(tuple(DTYPES)), _log(rng, 64, 1 << 20),
                  rng.random() < 0.5, rng.random() < 0.5)
    elif op == "verify":
        vocab = _log(rng, 50, 150000)
        c = _verify("", _log(rng, 1, min(256, max(1, 24_000_000 // vocab))), rng.randint(1, 8), vocab, rng.choice((0, 0, 1, 64)), ragged)
    else:
        dim, kv = rng.choice((32, 64, 128)), rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 3, 4, 7, 8))
        dtype, page = rng.choice(("bf16", "fp16")), rng.choice((16, 32, 64, 128))
        if op == "append":
            batch = _log(rng, 1, 128)
            new = _log(rng, 1, max(1, min(2048, 8192 // batch)))
            c = _append("", batch, rng.choice((0, 1, max(1, new // 4))), new, heads, kv, dim,
                        rng.choice((dim, dim // 2, dim - 8, 0)), rng.choice(("half", "interleaved")),
                        rng.choice(("fp32", dtype)), dtype, page, _log(rng, 1, 4096) - 1, new + _log(rng, 1, 1024),
                        rng.random() < 0.5, ragged)
        else:
            batch, new = _log(rng, 1, 128), rng.randint(1, 6)
            prefix = _log(rng, 1, 16384) - 1
            longest = new + _log(rng, 1, max(1, min(2042, 262144 // batch)))
            low = rng.choice((0, 1, new))
            while 4 * dim * heads * batch * new * (prefix + longest) > 100e9:
                prefix //= 2                            # no dearer than the largest listed case
            c = _attend("", batch, low, new, heads, kv, dim, dtype, page, prefix, longest, ragged)
    del c["name"]
    return c


def _lengths(c):
    """(new tokens, own cached tokens) of each sequence: of the case, whatever the seed."""
    r = random.Random(c["ragged"])
    new = [r.randint(c.get("low", 1), c["new"]) for _ in range(c["batch"])]
    new[r.randrange(len(new))] = c["new"]
    if "longest" not in c:
        return new, None
    own_len = [r.randint(n, c["longest"]) for n in new]
    own_len[0] = c["longest"]
    return new, own_len


# ------------------------------------------------------------------------------------------------ the rotation's plan
def _frequencies(rot, scaling, base=10000.0, factor=8.0, original=4096, slow=1.0, fast=32.0):
    """Turns a position of each pair, in 64 bits, and the magnitude of the rotated part."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"), -2.0 * i / rot) / (2.0 * math.pi)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        keep = ((f * original - slow) / (fast - slow)).clamp(0.0, 1.0)
        return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rotate(x, pos, f, m, rot, layout, sign):
    """x [rows, heads, dim] rotated in 32 bits; pos [rows]."""
    if rot == 0:
        return x.float()
    turns = pos.double()[:, None] * f
    angle = (turns - torch.round(turns)) * (2.0 * math.pi)
    c, s = (torch.cos(angle) * m).float()[:, None, :], (torch.sin(angle) * (m * sign)).float()[:, None, :]
    x = x.float()
    if layout == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


# ------------------------------------------------------------------------------------------------ inputs
def _batch(c, g):
    """start, len, pages, prefix_pages and the number of pages: every page number once, in no order."""
    new, length = _lengths(c)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    page = c["page"]
    most, first = -(-c["longest"] // page), -(-c["prefix"] // page)
    pages = first + most * c["batch"] + 1
    order = torch.randperm(pages, generator=g, device="cuda").int()
    return {"start": torch.tensor(start, dtype=torch.int32).cuda(), "len": torch.tensor(length, dtype=torch.int32).cuda(),
            "prefix_pages": order[: max(first, 1)].clone(), "pages": order[first: first + most * c["batch"]].reshape(c["batch"], most).clone(),
            "count": pages, "rows": start[-1] + 3}      # three rows behind the last sequence, as a padded batch has


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[dtype])

    t = {}
    if c["op"] == "rope":
        ld = (c["heads"] + 2) * c["dim"] if c["packed"] else c["heads"] * c["dim"]
        t["x"] = normal((c["rows"], ld), c["dtype"])
        t["y"] = torch.zeros((c["rows"], c["heads"], c["dim"]), dtype=DTYPES[c["dtype"]], device="cuda")
        t["pos"] = torch.randint(0, c["far"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
    elif c["op"] == "verify":
        new, _ = _lengths(c)
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        rows, v = start[-1] + 2, c["vocab"]
        z = torch.randn((rows, v), generator=g, device="cuda") * 2.5
        t["p"] = torch.zeros((rows, v + c["pad"]), device="cuda")
        t["q"] = torch.zeros((rows, v + c["pad"]), device="cuda")
        t["p"][:, :v] = torch.softmax(z, 1)
        z += torch.randn((rows, v), generator=g, device="cuda") * 0.7
        t["q"][:, :v] = torch.softmax(z, 1)
        z -= torch.log(-torch.log(torch.rand((rows, v), generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
        t["draft"] = z.argmax(1).int()                  # a draw from q
        t["u"] = torch.rand((rows,), generator=g, device="cuda")
        t["start"] = torch.tensor(start, dtype=torch.int32).cuda()
        t["tokens"] = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
        t["accepted"] = torch.full((c["batch"],), -7, dtype=torch.int32, device="cuda")
        t["rows"] = rows
    else:
        t = _batch(c, g)
        rows, hq, hk, d = t["rows"], c["q_heads"], c["kv_heads"], c["dim"]
        t["k_cache"] = normal((t["count"], hk, c["page"], d), c["dtype"])
        t["v_cache"] = normal((t["count"], hk, c["page"], d), c["dtype"])
        if c["op"] == "attend":
            t["q"] = normal((rows, hq, d), c["dtype"], 2.0)
            t["out"] = torch.zeros((rows, hq, d), dtype=DTYPES[c["dtype"]], device="cuda")
        else:
            if c["packed"]:
                t["qkv"] = normal((rows, (hq + 2 * hk) * d), c["src"])
            else:
                t["q"], t["k"], t["v"] = (normal((rows, h * d), c["src"]) for h in (hq, hk, hk))
            t["q_out"] = torch.zeros((rows, hq, d), dtype=DTYPES[c["dtype"]], device="cuda")
    t["case"] = c
    if own:
        return _own_state(t)
    if c["op"] in ("rope", "append"):
        t["plan"] = _frequencies(c["rot"], c.get("scaling", "none")) if c["rot"] else (None, 1.0)
    return t


# ------------------------------------------------------------------------------------------------ the plain forms
def _sources(s, c):
    if not c["packed"]:
        return s["q"], s["k"], s["v"]
    a, b = c["q_heads"] * c["dim"], (c["q_heads"] + c["kv_heads"]) * c["dim"]
    return s["qkv"][:, :a], s["qkv"][:, a:b], s["qkv"][:, b:]


def _owner(start, rows):
    """Each row's sequence (the batch's size behind the last one) and its place in it."""
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(start[1:].contiguous(), t.int(), right=True)
    return t, b


def _run_rope(s, c):
    x = s["x"][:, : c["heads"] * c["dim"]].reshape(c["rows"], c["heads"], c["dim"])
    f, m = s["plan"]
    y = _rotate(x, s["pos"], f, m, c["rot"], c["layout"], -1.0 if c["inverse"] else 1.0)
    return {"y": y.to(x.dtype)}


def _run_append(s, c):
    t, b = _owner(s["start"], s["rows"])
    n = int(s["rows"]) - 3
    t, b = t[:n], b[:n]
    new = s["start"][1:] - s["start"][:-1]
    own_at = s["len"][b] - new[b] + t - s["start"][b]
    pos = own_at + c["prefix"]
    q, k, v = (x[:n].reshape(n, -1, c["dim"]) for x in _sources(s, c))
    f, m = s["plan"]
    dtype = s["k_cache"].dtype
    s["q_out"][:n] = _rotate(q, pos, f, m, c["rot"], c["layout"], 1.0).to(dtype)
    page, slot = s["pages"][b, own_at // c["page"]].long(), (own_at % c["page"]).long()
    s["k_cache"][page, :, slot] = _rotate(k, pos, f, m, c["rot"], c["layout"], 1.0).to(dtype)
    s["v_cache"][page, :, slot] = v.to(dtype)
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_attend(s, c):
    d, hk, page, size, most = c["dim"], c["kv_heads"], c["page"], c["batch"], c["new"]
    group, rows = c["q_heads"] // hk, s["rows"]
    new = s["start"][1:] - s["start"][:-1]
    j = torch.arange(most, device="cuda")
    at = (s["start"][:-1, None] + j).clamp(max=rows - 1).long()                     # [batch, most]
    q = s["q"][at].float().reshape(size, most, hk, group, d)
    first = s["prefix_pages"].long()

    def shared(x):
        return x[first].float().transpose(0, 1).reshape(hk, -1, d)[:, : c["prefix"]]

    def each(x, keep):
        x = x[s["pages"].long()].float().transpose(1, 2).reshape(size, hk, -1, d)
        return torch.where(keep[:, None, :, None], x, torch.zeros((), device="cuda"))

    own_at = torch.arange(s["pages"].shape[1] * page, device="cuda")
    held = own_at < s["len"][:, None]
    sees = own_at < (s["len"] - new)[:, None, None] + j[None, :, None] + 1           # [batch, most, keys]
    scale = 1.0 / math.sqrt(d)
    flat = q.permute(2, 0, 1, 3, 4).reshape(hk, -1, d)
    a = torch.matmul(flat, shared(s["k_cache"]).transpose(1, 2)) * scale             # [kv heads, batch * most * group, prefix]
    e = torch.matmul(q.transpose(1, 2).reshape(size, hk, most * group, d), each(s["k_cache"], held).transpose(2, 3)) * scale
    e = e.reshape(size, hk, most, group, -1).masked_fill(~sees[:, None, :, None, :], -math.inf)
    e = e.permute(1, 0, 2, 3, 4).reshape(hk, size * most * group, -1)
    top = e.amax(-1, keepdim=True)
    if c["prefix"]:
        top = torch.maximum(top, a.amax(-1, keepdim=True))
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    a, e = torch.exp(a - top), torch.exp(e - top)
    total = a.sum(-1, keepdim=True) + e.sum(-1, keepdim=True)
    o = torch.matmul(a, shared(s["v_cache"]))
    e = e.reshape(hk, size, most * group, -1).transpose(0, 1)
    o = o + torch.matmul(e, each(s["v_cache"], held)).transpose(0, 1).reshape(hk, size * most * group, d)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(hk, size, most, group, d).permute(1, 2, 0, 3, 4).reshape(size, most, c["q_heads"], d)
    real = j[None, :] < new[:, None]
    s["out"][at[real]] = o[real].to(s["out"].dtype)
    return {"out": s["out"]}


def _run_verify(s, c):
    start, v, rows = s["start"].long(), c["vocab"], s["rows"]
    new = start[1:] - start[:-1]
    j = torch.arange(c["new"], device="cuda")
    at = (start[:-1, None] + j).clamp(max=rows - 1)
    draft = s["draft"][at].long()
    p, q, u = s["p"][at, draft].double(), s["q"][at, draft].double(), s["u"][at].double()
    good = (u * q < p) & (j < new[:, None] - 1)
    taken = good.long().cumprod(1).sum(1)
    row = (start[:-1] + taken).clamp(max=rows - 1)
    last = taken >= new - 1
    p = s["p"][row, :v].double()
    w = (p - torch.where(last[:, None], 0.0, s["q"][row, :v].double())).clamp(min=0.0)
    total = w.cumsum(1)
    r = s["u"][(start[1:] - 1).clamp(min=0)].double()[:, None]
    token = (total > r * total[:, -1:]).int().argmax(1)
    real = j < new[:, None]
    told = torch.where(j < taken[:, None], draft, torch.where(j == taken[:, None], token[:, None], -1)).int()
    s["tokens"][at[real]] = told[real]
    s["accepted"].copy_(taken)
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


def run(state):
    c = state["case"]
    if own:
        return state["call"]()
    return {"rope": _run_rope, "append": _run_append, "attend": _run_attend, "verify": _run_verify}[c["op"]](state, c)


# ------------------------------------------------------------------------------------------------ the framework's calls
class _Memory:
    """A device buffer's memory for torch.as_tensor."""

    def __init__(self, pointer, count, keep):
        self.__cuda_array_interface__ = {"data": (pointer, False), "shape": (count,), "typestr": "<f4", "version": 3}
        self.keep = keep


def _view(handle, like, keep):
    from zillaphp_b200 import native
    words = max(1, (like.numel() * like.element_size() + 3) // 4)
    flat = torch.as_tensor(_Memory(native.load().zilla_buffer_ptr(handle), words, keep), device="cuda")
    return flat.view(like.dtype)[: like.numel()].view(like.shape)


def _own_state(t):
    """The same inputs in the framework's buffers, and the call that a program makes on them."""
    import ctypes
    from zillaphp_b200 import autograd, native
    from zillaphp_b200.kv import PagedKv
    native.load().zilla_set_stream(ctypes.c_void_p(1))       # the legacy default stream, on which torch works here
    be, c = autograd.backend(), t["case"]
    s, ids = {}, {}
    for name in [k for k, v in t.items() if isinstance(v, torch.Tensor) and not k.endswith("_cache")]:
        x = t.pop(name)
        held = autograd.Tensor.empty(((x.numel() * x.element_size() + 3) // 4,))
        s[name], ids[name] = _view(held.buf, x, held), held.buf
        s[name].copy_(x)
        del x
    code = CODES[c["dtype"]] if "dtype" in c else 0
    layout = 1 if c.get("layout") == "interleaved" else 0
    table = 0
    if c.get("rot"):
        s["table"] = autograd.Tensor.empty((c["rot"] + 2,))
        table = s["table"].buf
        be.ropeTableDev(table, c["rot"], 10000.0, SCALINGS[c.get("scaling", "none")], 8.0, 4096, 1.0, 32.0)
    if c["op"] == "rope":
        wide, ld = c["heads"] * c["dim"], s["x"].shape[1]
        args = (ids["x"], 0, ld, ids["y"], 0, wide, ids["pos"], table, code, c["rows"], c["heads"], c["dim"], c["rot"],
                layout, 1 if c["inverse"] else 0)
        result = {"y": s["y"]}

        def call():
            be.ropeDev(*args)
            return result
    elif c["op"] == "verify":
        args = (ids["p"], s["p"].shape[1], ids["q"], s["q"].shape[1], ids["draft"], ids["u"], ids["start"],
                ids["tokens"], ids["accepted"], c["batch"], t["rows"], c["vocab"])
        result = {"tokens": s["tokens"], "accepted": s["accepted"]}

        def call():
            be.draftVerifyDev(*args)
            return result
    else:
        kv = s["kv"] = PagedKv(t["count"], c["page"], c["kv_heads"], c["dim"], c["dtype"])
        for name, handle in (("k_cache", kv.k_id), ("v_cache", kv.v_id)):
            x = t.pop(name)
            s[name] = _view(handle, x, kv)
            s[name].copy_(x)
            del x
        most = s["pages"].shape[1]
        if c["op"] == "attend":
            work = kv.attend_work(c["batch"], t["rows"], c["q_heads"], c["prefix"], c["new"], c["longest"])
            s["work"] = autograd.Tensor.empty((max(1, work),))
            args = (ids["q"], ids["out"], ids["start"], ids["len"], ids["pages"], ids["prefix_pages"], c["batch"], t["rows"],
                    c["q_heads"], most, c["prefix"], c["new"], c["longest"], 1.0 / math.sqrt(c["dim"]), s["work"].buf)
            result = {"out": s["out"]}

            def call():
                kv.attend(*args)
                return result
        else:
            wq, wk = c["q_heads"] * c["dim"], c["kv_heads"] * c["dim"]
            if c["packed"]:
                x, ld = ids["qkv"], wq + 2 * wk
                src = (x, 0, ld, x, wq, ld, x, wq + wk, ld)
            else:
                src = (ids["q"], 0, wq, ids["k"], 0, wk, ids["v"], 0, wk)
            args = (CODES[c["src"]], *src, ids["q_out"], ids["start"], ids["len"], ids["pages"], c["batch"], t["rows"],
                    c["q_heads"], most, c["prefix"], table, c["rot"], layout)
            result = {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}

            def call():
                kv.append(*args)
                return result
    s["case"], s["call"] = c, call
    return s


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if c["op"] == "rope":
        n = c["rows"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * size[c["dtype"]] + 4 * c["rows"], "flops": 3 * c["rows"] * c["heads"] * c["rot"]}
    new, length = _lengths(c)
    rows = sum(new)
    if c["op"] == "verify":
        # one row of p each; one of q where a draft fails: about 0.3 of the drafts do, by these inputs
        fails = sum(1.0 - 0.7 ** (n - 1) for n in new)
        return {"bytes": 4 * c["vocab"] * (c["batch"] + fails) + 20 * rows, "flops": 3 * c["vocab"] * c["batch"]}
    wide = (c["q_heads"] + 2 * c["kv_heads"]) * c["dim"]
    if c["op"] == "append":
        return {"bytes": rows * wide * (size[c["src"]] + size[c["dtype"]]), "flops": 3 * rows * wide}
    keys = c["prefix"] + sum(length)
    seen = rows * c["prefix"] + sum(max(0, own_len - n + j + 1) for n, own_len in zip(new, length) for j in range(n))
    return {"bytes": 2 * (2 * keys * c["kv_heads"] * c["dim"] + 2 * rows * c["q_heads"] * c["dim"]),
            "flops": 4 * c["dim"] * c["q_heads"] * seen}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _turn(x, pos, c):
    """One token's heads [heads, dim] in 64 bits, rotated as complex numbers at the given position."""
    rot = c["rot"]
    if not rot:
        return x
    rate = []
    for i in range(rot // 2):
        base = 10000.0 * (8.0 ** (rot / (rot - 2.0)) if c.get("scaling") == "base" and rot > 2 else 1.0)
        w = base ** (-2.0 * i / rot)
        if c.get("scaling") == "linear":
            w /= 8.0
        if c.get("scaling") == "parts":
            ramp = min(1.0, max(0.0, (4096.0 * w / (2.0 * math.pi) - 1.0) / 31.0))
            w = (1.0 - ramp) * w / 8.0 + ramp * w
        rate.append(w)
    m = 0.1 * math.log(8.0) + 1.0 if c.get("scaling") == "parts" else 1.0
    angle = torch.outer(pos.double(), torch.tensor(rate, dtype=torch.float64, device="cuda"))
    if c.get("inverse"):
        angle = -angle
    z = torch.polar(torch.full_like(angle, m), angle)[:, None, :]
    y = x.clone()
    if c["layout"] == "half":
        w = torch.complex(x[..., : rot // 2], x[..., rot // 2: rot]) * z
        y[..., : rot // 2], y[..., rot // 2: rot] = w.real, w.imag
    else:
        w = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * z
        y[..., 0:rot:2], y[..., 1:rot:2] = w.real, w.imag
    return y


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "rope":
        x = s["x"][:, : c["heads"] * c["dim"]].double().reshape(c["rows"], c["heads"], c["dim"])
        return {"y": _turn(x, s["pos"], c)}
    new, length = _lengths(c)
    if c["op"] == "verify":
        return None                                      # whole numbers: the plain form's have to be met
    page, d, group = c["page"], c["dim"], c["q_heads"] // c["kv_heads"]
    if c["op"] == "append":
        q, k, v = _sources(s, c)
        out, kc, vc = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
        table, row = s["pages"].tolist(), 0
        for b, (n, held) in enumerate(zip(new, length)):
            at = torch.arange(held - n, held, device="cuda")
            where = torch.tensor([table[b][i // page] for i in range(held - n, held)], dtype=torch.long, device="cuda")
            pos = at + c["prefix"]
            out[row: row + n] = _turn(q[row: row + n].double().reshape(n, -1, d), pos, c)
            kc[where, :, at % page] = _turn(k[row: row + n].double().reshape(n, -1, d), pos, c)
            vc[where, :, at % page] = v[row: row + n].double().reshape(n, -1, d)
            row += n
        return {"q": out, "k_cache": kc, "v_cache": vc}
    if c["q_heads"] * sum(new) * (c["prefix"] + c["longest"]) * c["dim"] > 1e11:
        return None
    out = s["out"].double()
    front = s["prefix_pages"].long()
    for h in range(c["kv_heads"]):
        k0 = s["k_cache"][front, h].double().reshape(-1, d)[: c["prefix"]]
        v0 = s["v_cache"][front, h].double().reshape(-1, d)[: c["prefix"]]
        row = 0
        for b, (n, held) in enumerate(zip(new, length)):
            mine = s["pages"][b].long()
            k1 = torch.cat((k0, s["k_cache"][mine, h].double().reshape(-1, d)[:held]))
            v1 = torch.cat((v0, s["v_cache"][mine, h].double().reshape(-1, d)[:held]))
            if n:
                x = torch.einsum("tgd,kd->tgk", s["q"][row: row + n, h * group: (h + 1) * group].double(), k1) / math.sqrt(d)
                last = c["prefix"] + held - n + torch.arange(n, device="cuda")
                x[torch.arange(k1.shape[0], device="cuda")[None, None, :].expand_as(x) > last[:, None, None]] = -math.inf
                out[row: row + n, h * group: (h + 1) * group] = torch.einsum("tgk,kd->tgd", torch.softmax(x, -1), v1)
            row += n
    return {"out": out}
