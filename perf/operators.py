"""The operators that serve many utterances of one voice from a paged K/V
cache: what is measured of them, and their plain forms.

A speaker's conditioning (1 speaker row + 375 prompt tokens in the T3 GGUF) is
the same for every utterance of a voice and for both rows of a CFG stream, so
its K/V is one shared prefix; each request's own tokens live in pages of a
common pool.  Four operators make that path:

  plan    block tables, slot maps and row maps of a batch, from the requests'
          lengths (t3b_op_kv_plan)
  append  the new tokens' K and V rows into their pages (t3b_op_kv_append)
  decode  attention of one query token per request over its prefix and its
          own pages (t3b_op_attention_shared)
  prompt  the same for a ragged batch of prompt chunks, causal over the own
          tokens (t3b_op_attention_shared_prompt)
"""
import ctypes
import importlib.util
import math
import os
import sys

import torch

own = False   # run(): False = the plain forms below, True = the framework's operators

DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 64 utterances in flight: every request gets one
        # token, one in sixteen of them a new page
        dict(name="plan-decode-64", op="plan", requests=64, page=16, blocks=128, admit=0, prompt=1, retire=0),
        # a step of a busy server: 200 utterances decode, 40 are admitted with
        # their text (up to 120 tokens), 16 slots give their pages back
        dict(name="plan-mixed-256", op="plan", requests=256, page=16, blocks=80, admit=40, prompt=120, retire=16),
        # a large admission wave: text of up to 200 tokens for 1000 requests
        dict(name="plan-wave-2048", op="plan", requests=2048, page=32, blocks=48, admit=1000, prompt=200, retire=100),
        # the K/V rows of 64 CFG streams' decode step (f32 from the QKV GEMV)
        dict(name="append-decode-128", op="append", type="f32", rows=128, kv_heads=16, dim=64, page=16, pad=0),
        # the text of a few utterances
        dict(name="append-text-1500", op="append", type="f32", rows=1500, kv_heads=16, dim=64, page=16, pad=64),
        # long prompts of a grouped-head model, rows cut out of a wider buffer
        dict(name="append-prompts-20001", op="append", type="bf16", rows=20001, kv_heads=8, dim=128, page=64, pad=256),
        # one utterance with CFG: two rows over the same voice (latency)
        dict(name="decode-one-cfg-stream", op="decode", type="f32", requests=2, prefixes=1, prefix=376, lo=88, hi=600,
             heads=16, kv_heads=16, dim=64, page=16),
        # 64 CFG streams of one voice, anywhere between their text and 1000 speech tokens
        dict(name="decode-64-cfg-streams", op="decode", type="f32", requests=128, prefixes=1, prefix=376, lo=88, hi=1088,
             heads=16, kv_heads=16, dim=64, page=16),
        # short answers behind a long shared prefix: the prefix is most of the arithmetic
        dict(name="decode-short-long-prefix", op="decode", type="bf16", requests=256, prefixes=1, prefix=4096, lo=1,
             hi=200, heads=32, kv_heads=8, dim=128, page=32),
        # the largest: four prefixes, long own contexts, bound by the own K/V
        dict(name="decode-long-own", op="decode", type="f16", requests=192, prefixes=4, prefix=8192, lo=500, hi=4000,
             heads=32, kv_heads=8, dim=128, page=64),
        # the text prompts of 16 utterances of two voices
        dict(name="prompt-text-16", op="prompt", type="f32", requests=16, prefixes=2, prefix=376, lo=20, hi=120, past=0,
             heads=16, kv_heads=16, dim=64, page=16),
        # long prompt chunks, some of them continuing an earlier chunk
        dict(name="prompt-chunks-8", op="prompt", type="bf16", requests=8, prefixes=1, prefix=1000, lo=300, hi=2000,
             past=700, heads=32, kv_heads=8, dim=128, page=64),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _layout(rng):
    kv = rng.choice([1, 2, 4, 8, 16])
    g = rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv <= 32])
    return dict(heads=kv * g, kv_heads=kv, dim=rng.choice([64, 128]), page=rng.choice([8, 16, 32, 64, 128]))


def draw(rng):
    op = rng.choice(["plan", "append", "decode", "decode", "prompt"])
    if op == "plan":
        n = _spread(rng, 1, 2048)
        admit = rng.randint(0, n // 2)
        return dict(op=op, requests=n, page=rng.choice([8, 16, 32, 64]), blocks=rng.randint(32, 64), admit=admit,
                    prompt=rng.randint(1, 200), retire=rng.randint(0, (n - admit) // 4))
    if op == "append":
        lay = _layout(rng)
        rows = _spread(rng, 1, 20001 * 1024 // (lay["kv_heads"] * lay["dim"]) if lay["kv_heads"] * lay["dim"] > 1024
                       else 20001)
        return dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), rows=rows, kv_heads=lay["kv_heads"],
                    dim=lay["dim"], page=lay["page"], pad=8 * rng.randint(0, 32))
    lay = _layout(rng)
    prefixes = rng.choice([1, 1, 2, 4])
    prefix = _spread(rng, 1, 8192 if op == "decode" else 2000)
    if op == "decode":
        case = dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), requests=prefixes * _spread(rng, 1, 192 // prefixes),
                    prefixes=prefixes, prefix=prefix, lo=1, hi=_spread(rng, 1, 4000), **lay)
        case["lo"] = rng.randint(1, case["hi"])
    else:
        case = dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), requests=prefixes * _spread(rng, 1, 16 // prefixes),
                    prefixes=prefixes, prefix=prefix, lo=1, hi=_spread(rng, 1, 2000), past=rng.choice([0, 0, 100, 700]),
                    **lay)
        case["lo"] = rng.randint(1, case["hi"])
    most = work(next(c for c in listed() if c["name"] == ("decode-long-own" if op == "decode" else "prompt-chunks-8")))
    while True:
        w = work(case)
        f = max(w["bytes"] / most["bytes"], w["flops"] / most["flops"])
        if f <= 1 or (case["requests"] == prefixes and case["hi"] == 1):
            return case
        if case["requests"] > prefixes:
            case["requests"] = prefixes * max(1, int(case["requests"] / prefixes / min(f, 2.0)))
        else:
            case["hi"] = max(1, case["hi"] // 2)
            case["lo"] = min(case["lo"], case["hi"])


def work(case):
    """Bytes and operations of one pass, at the mean of the drawn lengths."""
    op, c = case["op"], case
    if op == "plan":
        n = c["requests"]
        decode = n - c["admit"] - c["retire"]
        rows = decode + c["admit"] * (c["prompt"] + 1) / 2
        taken = decode / c["page"] + c["admit"] * ((c["prompt"] + 1) / 2 / c["page"] + 0.5)
        given = c["retire"] * c["blocks"] / 4
        # lengths, new tokens and releases in, row starts and lengths out; an id read and
        # written per page that moves; request, position and slot per row
        return {"bytes": 4.0 * (5 * n + 2 * taken + 2 * given + 3 * rows), "flops": 0.0}
    if op == "append":
        src = 4 if c["type"] == "f32" else 2
        return {"bytes": float(c["rows"]) * (2 * c["kv_heads"] * c["dim"] * (src + 2) + 4), "flops": 0.0}
    q = 4 if c["type"] == "f32" else 2
    mean = (c["lo"] + c["hi"]) / 2
    kv = 2 * 2 * c["kv_heads"] * c["dim"]                      # bytes of a token's K and V
    pre = sum(_prefix_lens(c))
    if op == "decode":
        n = c["requests"]
        keys = pre / c["prefixes"] + mean
        return {"bytes": kv * (pre + n * mean) + 2 * n * c["heads"] * c["dim"] * q,
                "flops": 4.0 * n * c["heads"] * c["dim"] * keys}
    rows = c["requests"] * mean
    keys = pre / c["prefixes"] + c["past"] / 2 + (mean + 1) / 2
    return {"bytes": kv * (pre + rows + c["requests"] * c["past"] / 2) + 2 * rows * c["heads"] * c["dim"] * q,
            "flops": 4.0 * rows * c["heads"] * c["dim"] * keys}


def _prefix_lens(c):
    """Lengths of the prefixes: the first has all of case["prefix"], the others end inside a page."""
    return [max(1, c["prefix"] - 37 * i) for i in range(c["prefixes"])]


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "plan":
        _prepare_plan(s, case, g)
    elif case["op"] == "append":
        _prepare_append(s, case, g)
    else:
        _prepare_attention(s, case, g)
    return s


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int32)


def _pages(tokens, page):
    return (tokens + page - 1) // page


def _prepare_plan(s, c, g):
    n, page, blocks = c["requests"], c["page"], c["blocks"]
    order = torch.randperm(n, generator=g, device=DEV)             # slots fill in no order
    kind = torch.zeros(n, dtype=torch.int32, device=DEV)
    kind[order[:c["admit"]]] = 1
    kind[order[c["admit"]:c["admit"] + c["retire"]]] = 2
    most = blocks * page - 1
    used = _ints(g, 1, most // 2, n)
    zero = torch.zeros_like(used)
    s["len"] = torch.where(kind == 0, used, zero)
    s["add"] = torch.where(kind == 0, 1 + zero, torch.where(kind == 1, _ints(g, 1, min(c["prompt"], most), n), zero))
    s["release"] = torch.where(kind == 2, used, zero)
    held = _pages(torch.where(kind == 1, zero, used), page)
    n_pages = n * blocks
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    at = torch.cumsum(held, 0) - held
    col = torch.arange(blocks, device=DEV)
    has = col[None] < held[:, None]
    s["table"] = torch.where(has, ids[(at[:, None] + col[None]).clamp(max=n_pages - 1)], -1).to(torch.int32)
    taken = held.sum()
    # the stack of free pages: the ids that no request holds, then room for those that come back
    s["free"] = torch.roll(ids, -int(taken))
    s["n_free"] = (n_pages - taken).to(torch.int32).reshape(1)
    s["n_free_out"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    s["rows"] = (n - c["admit"] - c["retire"]) + c["admit"] * c["prompt"]      # what the host knows: a bound
    for k in ("row_req", "row_pos", "slots"):
        s[k] = torch.empty(max(1, s["rows"]), dtype=torch.int32, device=DEV)
    s["row_start"] = torch.empty(n + 1, dtype=torch.int32, device=DEV)
    s["len_out"] = torch.empty(n, dtype=torch.int32, device=DEV)


def _prepare_append(s, c, g):
    rows, width = c["rows"], c["kv_heads"] * c["dim"]
    n_pages = _pages(rows, c["page"]) + 7
    store = torch.bfloat16 if c["type"] == "bf16" else torch.float16
    wide = torch.randn(2, rows, width + c["pad"], generator=g, device=DEV, dtype=DT[c["type"]])
    s["k_new"], s["v_new"] = wide[0, :, :width], wide[1, :, :width]
    shape = (n_pages, c["kv_heads"], c["page"], c["dim"])
    s["k"] = torch.randn(shape, generator=g, device=DEV, dtype=store)
    s["v"] = torch.randn(shape, generator=g, device=DEV, dtype=store)
    # pages in no order, the rows of a page one after the other; one row in 32 is padding
    pages = torch.randperm(n_pages, generator=g, device=DEV)
    s["spare"] = pages[-1] * c["page"]                           # a slot that no row goes to
    pages = pages[:_pages(rows, c["page"])]
    slots = (pages[:, None] * c["page"] + torch.arange(c["page"], device=DEV)[None]).reshape(-1)[:rows]
    s["slots"] = torch.where(torch.arange(rows, device=DEV) % 32 == 31, -1, slots).to(torch.int32)


def _prepare_attention(s, c, g):
    n, G, page = c["requests"], c["prefixes"], c["page"]
    kv, dim = c["kv_heads"], c["dim"]
    store = torch.bfloat16 if c["type"] == "bf16" else torch.float16
    pre_blocks = _pages(c["prefix"], page)
    own_most = c["hi"] + c.get("past", 0)
    blocks = _pages(own_most, page)
    n_pages = G * pre_blocks + n * blocks
    shape = (n_pages, kv, page, dim)
    s["k"] = torch.randn(shape, generator=g, device=DEV, dtype=store)
    s["v"] = torch.randn(shape, generator=g, device=DEV, dtype=store)
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    s["prefix_table"] = ids[:G * pre_blocks].reshape(G, pre_blocks).contiguous()
    s["table"] = ids[G * pre_blocks:].reshape(n, blocks).contiguous()
    s["prefix_len"] = torch.tensor(_prefix_lens(c), dtype=torch.int32, device=DEV)
    s["prefix_start"] = torch.arange(G + 1, dtype=torch.int32, device=DEV) * (n // G)
    if c["op"] == "decode":
        s["len"], rows = _ints(g, c["lo"], c["hi"], n), n
    else:
        # chunk lengths spread evenly over lo .. hi, in an order of the seed's: the row count is the case's
        even = [c["lo"] + (c["hi"] - c["lo"]) * (2 * i + 1) // (2 * n) for i in range(n)]
        rows = sum(even)
        new = torch.tensor(even, dtype=torch.int32, device=DEV)[torch.randperm(n, generator=g, device=DEV)]
        past = _ints(g, 0, c["past"], n)
        s["len"], s["add"] = past + new, new
        s["row_start"] = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), torch.cumsum(new, 0).to(torch.int32)])
    s["rows"] = rows
    s["q"] = torch.randn(rows, c["heads"] * dim, generator=g, device=DEV, dtype=DT[c["type"]])
    s["out"] = torch.empty_like(s["q"])


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "append": _append, "decode": _decode, "prompt": _prompt}[state["case"]["op"]](state)


def _plan(s):
    page = s["case"]["page"]
    ln, add, rel, table, free, n_free = s["len"], s["add"], s["release"], s["table"], s["free"], s["n_free"]
    n, blocks = table.shape
    back = _pages(rel, page)                                    # pages that come back, on top of the stack
    back_at = torch.cumsum(back, 0) - back
    col = torch.arange(blocks, device=DEV)[None]
    stack = free.clone()
    ends = torch.where(col < back[:, None], n_free + back_at[:, None] + col, -1).reshape(-1)
    stack = torch.cat([stack, stack[:1]])                       # one place that nothing reads takes the rest
    stack[torch.where(ends < 0, free.numel(), ends)] = table.reshape(-1)
    stack = stack[:-1]
    top = n_free + back.sum()
    held, need = _pages(ln, page), _pages(ln + add, page)
    take = need - held
    take_at = torch.cumsum(take, 0) - take
    fresh = (col >= held[:, None]) & (col < need[:, None])
    pick = top - 1 - (take_at[:, None] + col - held[:, None])
    table = torch.where(fresh, stack[torch.where(fresh, pick, 0)], table)
    row_start = torch.cat([torch.zeros_like(add[:1]), torch.cumsum(add, 0).to(torch.int32)])
    row = torch.arange(s["row_req"].numel(), device=DEV, dtype=torch.int32)
    live = row < row_start[-1]
    req = torch.searchsorted(row_start[1:], row, right=True).clamp(max=n - 1)
    pos = ln[req] + row - row_start[req]
    slot = table[req, torch.where(live, pos // page, 0)] * page + pos % page
    pad = torch.full_like(row, -1)
    return dict(table=table, free=stack, n_free=(top - take.sum()).to(torch.int32), row_start=row_start,
                row_req=torch.where(live, req.to(torch.int32), pad), row_pos=torch.where(live, pos, pad),
                slots=torch.where(live, slot, pad), len=ln + add)


def _append(s):
    c, slots = s["case"], s["slots"].long()
    live = slots >= 0
    at = torch.where(live, slots, s["spare"])                    # padding rewrites what the spare slot holds
    page, off = at // c["page"], at % c["page"]
    shape = (c["rows"], c["kv_heads"], c["dim"])
    for name in ("k", "v"):
        new = s[name + "_new"].reshape(shape).to(s[name].dtype)
        s[name][page, :, off] = torch.where(live[:, None, None], new, s[name][page, :, off])
    return dict(k=s["k"], v=s["v"])


def _keys(pool, table):
    """[tables][kv heads][tokens][dim] in 32 bits of the pages that each row of `table` names."""
    t, b = table.shape
    x = pool[table.long()]                                       # [tables][blocks][kv heads][page][dim]
    return x.permute(0, 2, 1, 3, 4).reshape(t, x.shape[2], b * x.shape[3], x.shape[4]).float()


def _joint(pre, post, v_pre, v_own, G):
    """softmax over the prefix's and the own scores together; the products with V."""
    m = torch.maximum(pre.amax(-1, keepdim=True), post.amax(-1, keepdim=True))
    e_pre, e_own = torch.exp(pre - m), torch.exp(post - m)
    total = e_pre.sum(-1, keepdim=True) + e_own.sum(-1, keepdim=True)
    n, kv, r, L = e_pre.shape
    per = n // G
    o = e_pre.reshape(G, per, kv, r, L).permute(0, 2, 1, 3, 4).reshape(G, kv, per * r, L) @ v_pre
    o = o.reshape(G, kv, per, r, -1).permute(0, 2, 1, 3, 4).reshape(n, kv, r, -1)
    return (o + e_own @ v_own) / total


def _scores(s, q):
    """Scores of q [requests][kv heads][rows][dim] over the prefix and over the own pages, unmasked."""
    c = s["case"]
    G, n = c["prefixes"], c["requests"]
    kv, dim, r = c["kv_heads"], c["dim"], q.shape[2]
    per = n // G
    scale = 1.0 / math.sqrt(dim)
    k_pre, v_pre = _keys(s["k"], s["prefix_table"]), _keys(s["v"], s["prefix_table"])
    k_own, v_own = _keys(s["k"], s["table"]), _keys(s["v"], s["table"])
    qg = q.reshape(G, per, kv, r, dim).permute(0, 2, 1, 3, 4).reshape(G, kv, per * r, dim)
    pre = (qg @ k_pre.transpose(-1, -2)) * scale
    off = torch.arange(pre.shape[-1], device=DEV)[None] >= s["prefix_len"][:, None]
    pre = pre.masked_fill(off[:, None, None], -math.inf)
    pre = pre.reshape(G, kv, per, r, -1).permute(0, 2, 1, 3, 4).reshape(n, kv, r, -1)
    return pre, (q @ k_own.transpose(-1, -2)) * scale, v_pre, v_own


def _decode(s):
    c = s["case"]
    n, kv, dim, g = c["requests"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    q = s["q"].float().reshape(n, kv, g, dim)
    pre, post, v_pre, v_own = _scores(s, q)
    off = torch.arange(post.shape[-1], device=DEV)[None] >= s["len"][:, None]
    post = post.masked_fill(off[:, None, None], -math.inf)
    return _joint(pre, post, v_pre, v_own, c["prefixes"]).reshape(n, -1).to(s["q"].dtype)


def _prompt(s):
    c = s["case"]
    n, kv, dim, g = c["requests"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    most = c["hi"]
    # the ragged rows, padded to [requests][most rows]
    col = torch.arange(most, device=DEV)
    at = (s["row_start"][:-1, None] + col[None]).clamp(max=s["rows"] - 1).long()
    q = s["q"].float()[at].reshape(n, most, kv, g, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, most * g, dim)
    pre, post, v_pre, v_own = _scores(s, q)
    # row j of a request stands at own position len - add + j and sees the positions up to its own
    pos = (s["len"] - s["add"])[:, None] + col[None]
    off = torch.arange(post.shape[-1], device=DEV)[None, None] > pos[..., None]
    off = off[:, None, :, None].expand(n, 1, most, g, -1).reshape(n, 1, most * g, -1)
    post = post.masked_fill(off, -math.inf)
    o = _joint(pre, post, v_pre, v_own, c["prefixes"])
    o = o.reshape(n, kv, most, g, dim).permute(0, 2, 1, 3, 4).reshape(n * most, -1)
    row = torch.arange(s["rows"], device=DEV, dtype=torch.int32)
    req = torch.searchsorted(s["row_start"][1:], row, right=True)
    return o[req * most + row - s["row_start"][req]].to(s["q"].dtype)


# --------------------------------------------------------------------------
# from the definition, in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None                                              # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            x = s[name].double()
            flat = x.permute(0, 2, 1, 3).reshape(-1, case["kv_heads"], case["dim"])      # by slot
            slots = s["slots"].long()
            flat[slots[slots >= 0]] = s[name + "_new"].double().reshape(case["rows"], case["kv_heads"], -1)[slots >= 0]
            out[name] = flat.reshape(x.shape[0], case["page"], case["kv_heads"], -1).permute(0, 2, 1, 3)
        return out
    n, kv, dim, heads, page = (case[k] for k in ("requests", "kv_heads", "dim", "heads", "page"))
    lens, starts = s["len"].tolist(), s["row_start"].tolist() if "row_start" in s else list(range(n + 1))
    pre_lens, per = s["prefix_len"].tolist(), n // case["prefixes"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)

    def tokens(pool, ids, count):
        """[kv heads][count][dim]: token t is row t % page of page ids[t // page]."""
        t = torch.arange(count, device=DEV)
        return pool[ids.long()[t // page], :, t % page].double().transpose(0, 1)

    for i in range(n):
        p, rows = i // per, starts[i + 1] - starts[i]
        k, v = (torch.cat([tokens(s[x], s["prefix_table"][p], pre_lens[p]), tokens(s[x], s["table"][i], lens[i])], 1)
                for x in "kv")
        q = s["q"][starts[i]:starts[i + 1]].double().reshape(rows, heads, dim).transpose(0, 1)
        # the last of the request's rows sees all keys, each one before it one fewer
        see = k.shape[1] - rows + 1 + torch.arange(rows, device=DEV)
        hide = torch.arange(k.shape[1], device=DEV)[None] >= see[:, None]
        for h in range(heads):
            w = (q[h] @ k[h * kv // heads].T / math.sqrt(dim)).masked_fill(hide, -math.inf).softmax(-1)
            out[starts[i]:starts[i + 1], h * dim:(h + 1) * dim] = w @ v[h * kv // heads]
    return out


# --------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------

def _package():
    """chatterbox.cpp_b200/ (a folder name with a dot) as the module chatterbox_cpp_b200."""
    name = "chatterbox_cpp_b200"
    if name not in sys.modules:
        root = os.path.join(os.getcwd(), "chatterbox.cpp_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(root, "__init__.py"),
                                                      submodule_search_locations=[root])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def _describe(s):
    """The C structs of a call, filled once as a decode loop keeps them for its buffers."""
    pkg, c = _package(), s["case"]
    type_of = {torch.float32: pkg.T3B_F32, torch.float16: pkg.T3B_F16, torch.bfloat16: pkg.T3B_BF16}
    p = lambda name: s[name].data_ptr()  # noqa: E731
    if c["op"] == "plan":
        d = pkg.KvPlan(n=c["requests"], page_size=c["page"], max_blocks=c["blocks"], rows_cap=s["rows"], len=p("len"),
                       add=p("add"), release=p("release"), free_pages=p("free"), free_cap=s["free"].numel(),
                       n_free=p("n_free"), n_free_out=p("n_free_out"), table=p("table"), row_start=p("row_start"),
                       row_req=p("row_req"), row_pos=p("row_pos"), slots=p("slots"), len_out=p("len_out"))
        return pkg, pkg.lib().t3b_op_kv_plan, ctypes.byref(d), d
    cache = pkg.PagedKv(k=p("k"), v=p("v"), dtype=type_of[s["k"].dtype], n_pages=s["k"].shape[0], n_kv_head=c["kv_heads"],
                        page_size=c["page"], head_dim=c["dim"])
    if c["op"] == "append":
        d = pkg.KvAppend(cache=cache, k=p("k_new"), v=p("v_new"), dtype=type_of[s["k_new"].dtype], rows=c["rows"],
                         stride=s["k_new"].stride(0), slots=p("slots"))
        return pkg, pkg.lib().t3b_op_kv_append, ctypes.byref(d), d
    d = pkg.SharedAttn(cache=cache, q=p("q"), out=p("out"), dtype=type_of[s["q"].dtype], n_head=c["heads"],
                       q_stride=s["q"].stride(0), out_stride=s["out"].stride(0), n=c["requests"], rows=s["rows"],
                       len=p("len"), table=p("table"), max_blocks=s["table"].shape[1], n_prefix=c["prefixes"],
                       prefix_start=p("prefix_start"), prefix_len=p("prefix_len"), prefix_table=p("prefix_table"),
                       prefix_max_blocks=s["prefix_table"].shape[1])
    if c["op"] == "prompt":
        d.row_start = p("row_start")
    size = pkg.lib().t3b_op_attention_shared_workspace(ctypes.byref(d))
    s["workspace"] = torch.empty(max(1, size), dtype=torch.uint8, device=DEV)
    d.workspace, d.workspace_bytes = p("workspace"), size
    f = pkg.lib().t3b_op_attention_shared_prompt if c["op"] == "prompt" else pkg.lib().t3b_op_attention_shared
    return pkg, f, ctypes.byref(d), d


def _own(s):
    if "call" not in s:
        s["call"] = _describe(s)
    pkg, f, d, _ = s["call"]
    pkg.check(f(d, torch.cuda.current_stream().cuda_stream))
    op = s["case"]["op"]
    if op == "plan":
        return dict(table=s["table"], free=s["free"], n_free=s["n_free_out"], row_start=s["row_start"],
                    row_req=s["row_req"], row_pos=s["row_pos"], slots=s["slots"], len=s["len_out"])
    return dict(k=s["k"], v=s["v"]) if op == "append" else s["out"]
