"""Cases of the paged key-value cache operators: what is timed, on which inputs, and the operators in plain form.

Three operators work on one cache of fixed-size pages ([pages, H_kv, page_size, D] for keys and for values, and a
page table of int32 [sequences, pages of a sequence]):

* append: new key and value rows go to the pages behind each sequence's length; the rotary position rotation is
  applied to the keys (and to the queries beside them) on the way.
* decode: attention of one new token per sequence over its pages, with grouped heads; optionally capped scores,
  a window of the last keys and a bias that falls with distance.
* tree: attention of a pack of draft tokens per sequence (each sees the whole prefix in the pages and its own
  ancestors in the pack).

With `own` false `run` computes them from elementary torch operations in 32 bits (angles in 64); with `own` true it
calls this package.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------- cases
def _append(name, mode, dtype, B, lo, hi, new_lo, new_hi, Hq, Hkv, D, page, rot, interleaved=False, layers=1, pack=0):
    return dict(name=name, op="append", mode=mode, dtype=dtype, B=B, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, Hq=Hq,
                Hkv=Hkv, D=D, page=page, rot=rot, interleaved=interleaved, layers=layers, pack=pack)


def _decode(name, dtype, B, lo, hi, Hq, Hkv, D, page, cap=0.0, window=0, alibi=False, lse=False):
    return dict(name=name, op="decode", dtype=dtype, B=B, lo=lo, hi=hi, Hq=Hq, Hkv=Hkv, D=D, page=page, cap=cap,
                window=window, alibi=alibi, lse=lse)


def _tree(name, dtype, B, lo, hi, p_lo, p_hi, Hq, Hkv, D, page, words=False):
    return dict(name=name, op="tree", dtype=dtype, B=B, lo=lo, hi=hi, p_lo=p_lo, p_hi=p_hi, Hq=Hq, Hkv=Hkv, D=D,
                page=page, words=words)


def listed():
    return [
        # one user's decode step, the row starts a new page: launch and host latency are all there is
        _append("append_token_b1", "token", "bf16", 1, 512, 512, 1, 1, 32, 8, 128, 16, 128),
        # a large decode batch far into its contexts: half of each head is rotated, neighbouring pairs
        _append("append_token_b256", "token", "fp16", 256, 2000, 130000, 1, 1, 32, 8, 128, 64, 64, interleaved=True),
        # the prompts of a batch written to the cache, queries rotated beside the keys
        _append("append_prompts", "rows", "bf16", 16, 0, 0, 17, 4096, 32, 8, 128, 64, 128),
        # after a verify pass: the accepted rows of 64 packs of 128 draft tokens, eight layers in one call
        _append("append_accepted", "accept", "bf16", 64, 100, 200, 1, 9, 32, 8, 128, 64, 0, layers=8, pack=128),
        # one user early in a conversation
        _decode("decode_b1_short", "bf16", 1, 300, 300, 32, 8, 128, 16),
        # 64 ragged sequences of 4096 to 8192 keys: the cache is read once from memory
        _decode("decode_b64_ragged", "bf16", 64, 4096, 8192, 32, 8, 128, 64),
        # one very long document: the work is split over its length
        _decode("decode_b1_long", "fp16", 1, 131072, 131072, 64, 8, 128, 128),
        # capped scores and a sliding window, small pages, the log-sum-exp handed on
        _decode("decode_b32_window_cap", "bf16", 32, 100, 9000, 16, 8, 128, 16, cap=50.0, window=1024, lse=True),
        # 32-bit cache, three query heads to a key head, pages that are no power of two, distance bias
        _decode("decode_b33_f32_alibi", "fp32", 33, 1, 4000, 12, 4, 64, 24, alibi=True),
        # the smallest verify pass: one pack of 17 draft tokens
        _tree("tree_b1_small", "bf16", 1, 512, 512, 17, 17, 32, 8, 128, 16, words=True),
        # a full verify batch: 64 packs of 128 over prefixes of 4096 to 8192 keys
        _tree("tree_b64_full", "bf16", 64, 4096, 8192, 128, 128, 32, 8, 128, 64),
        # 32-bit inputs, small heads, odd packs and pages
        _tree("tree_b5_f32", "fp32", 5, 0, 1500, 1, 65, 12, 4, 64, 24),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "tree"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 3, 4, 7, 8, 16])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128, 256])
    e = 4 if dtype == "fp32" else 2
    per_key = 2 * Hkv * D * e
    if op == "append":
        mode = rng.choice(["token", "rows", "accept"])
        rot = rng.choice([0, D // 2, D, D])
        B = _log(rng, 1, 256)
        if mode == "token":
            return _append("", mode, dtype, B, 0, _log(rng, 16, 100000), 1, 1, Hkv * G, Hkv, D, page, rot,
                           rng.random() < 0.5)
        if mode == "rows":
            B = min(B, 40)
            rows = max(B, min(16384, (1 << 27) // (per_key * (1 + G // 2))))
            return _append("", mode, dtype, B, 0, rng.choice([0, 1, 777]), 0, max(1, _log(rng, 1, 2 * rows // B)),
                           Hkv * G, Hkv, D, page, rot, rng.random() < 0.5)
        layers = rng.choice([1, 2, 5])
        return _append("", mode, dtype, B, 0, 300, 0, _log(rng, 1, 16), Hkv * G, Hkv, D, page, rot,
                       rng.random() < 0.5, layers, _log(rng, 17, 128))
    if op == "decode":
        hi = _log(rng, 1, 131072)
        B = max(1, min(_log(rng, 1, 256), (1 << 30) // (per_key * hi)))
        return _decode("", dtype, B, rng.choice([0, 1, max(1, hi // 3), hi]) if hi > 1 else 1, hi, Hkv * G, Hkv, D, page,
                       rng.choice([0.0, 0.0, 30.0]), rng.choice([0, 0, _log(rng, 1, hi + 1)]), rng.random() < 0.25,
                       rng.random() < 0.5)
    p_hi = _log(rng, 1, 300)
    hi = _log(rng, 16, 16384)
    B = _log(rng, 1, 64)
    most = 2e10 if dtype == "fp32" else 2e11
    B = max(1, min(B, int(most / (4.0 * Hkv * G * D * p_hi * (hi + p_hi))), (1 << 30) // (per_key * hi)))
    return _tree("", dtype, B, rng.choice([0, hi // 4, hi]), hi, rng.choice([1, p_hi]), p_hi, Hkv * G, Hkv, D, page,
                 p_hi <= 64 and rng.random() < 0.5)


def _rng(case, what):
    return random.Random("%s %s" % (what, sorted((k, v) for k, v in case.items() if k != "name")))


def _spread(rng, n, lo, hi):
    """n lengths of [lo, hi], over their logarithm where they span more than a factor of ten."""
    if hi <= 10 * max(lo, 1):
        return [rng.randint(lo, hi) for _ in range(n)]
    return [min(hi, max(lo, _log(rng, max(lo, 1), hi) if rng.random() < 0.9 else lo)) for _ in range(n)]


def _plan(case):
    """What the host knows of a case: lengths, new rows or packs, parents."""
    B = case["B"]
    lens = _spread(_rng(case, "length"), B, case["lo"], case["hi"])
    if case["op"] == "append":
        new = _spread(_rng(case, "new"), B, case["new_lo"], case["new_hi"])
        return dict(lens=lens, new=new, rows=[case["pack"]] * B if case["mode"] == "accept" else new)
    if case["op"] == "decode":
        return dict(lens=lens, rows=[1] * B)
    rng = _rng(case, "pack")
    packs = _spread(rng, B, case["p_lo"], case["p_hi"])
    return dict(lens=lens, rows=packs, parents=[[-1] + [rng.randrange(max(0, i - 24), i) for i in range(1, p)] for p in packs])


def _depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def work(case):
    plan = _plan(case)
    e = 4 if case["dtype"] == "fp32" else 2
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    key = 2 * Hkv * D * e
    if case["op"] == "append":
        n = sum(plan["new"])
        q = 0 if case["mode"] == "accept" or not case["rot"] else Hq * D * e
        return {"bytes": 2 * n * (case["layers"] * key + q) + 12 * case["B"],
                "flops": 3 * n * case["rot"] * (case["layers"] * Hkv + (Hq if q else 0))}
    if case["op"] == "decode":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in plan["lens"])
        return {"bytes": seen * key + 2 * case["B"] * Hq * D * e + 4 * seen // case["page"], "flops": 4 * Hq * D * seen}
    pairs = sum(p * s + sum(_depths(t)) + p for p, s, t in zip(plan["rows"], plan["lens"], plan["parents"]))
    keys, rows = sum(plan["lens"]) + sum(plan["rows"]), sum(plan["rows"])
    return {"bytes": keys * key + 2 * rows * Hq * D * e, "flops": 4 * Hq * D * pairs}


# --------------------------------------------------------------------------------------------------- inputs
def _inv_freq(rot, dev):
    return (1.0 / (10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))).float().to(dev)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    dtype = _TYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    plan = _plan(case)
    B, Hq, Hkv, D, ps = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))

    def values(*shape, scale=1.0):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, scale, generator=g)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    grown = [n + m for n, m in zip(plan["lens"], plan["new"])] if case["op"] == "append" else plan["lens"]
    width = max(1, max(-(-n // ps) for n in grown))
    if case["op"] == "append" and case["mode"] == "token":
        # only the page that takes the new row matters: the long contexts before it share the pool's pages
        pages = 2 * B + 8
        table = torch.randint(0, B + 8, (B, width), device=dev, generator=g, dtype=torch.int32)
        last = ints([n // ps for n in plan["lens"]]).long()
        table[torch.arange(B, device=dev), last] = (torch.randperm(B, device=dev, generator=g) + B + 8).int()
    else:
        pages = B * width + 3 if B * width < 4096 else sum(-(-n // ps) for n in grown) + 3
        table = torch.zeros((B, width), dtype=torch.int32, device=dev)
        order = torch.randperm(pages, device=dev, generator=g).int()
        at = 0
        for b, n in enumerate(grown):
            m = -(-n // ps)
            table[b, :m] = order[at:at + m]
            at += m
    layers = case.get("layers", 1)
    kp = [values(pages, Hkv, ps, D) for _ in range(layers)]
    vp = [values(pages, Hkv, ps, D) for _ in range(layers)]
    total = sum(plan["rows"])
    cu = [0]
    for r in plan["rows"]:
        cu.append(cu[-1] + r)
    st = dict(case=case, plan=plan, cu=cu, k_pages=kp, v_pages=vp, table=table, lens=ints(plan["lens"]))
    if case["op"] == "append":
        st["k"] = [values(max(total, 1), Hkv, D) for _ in range(layers)]
        st["v"] = [values(max(total, 1), Hkv, D) for _ in range(layers)]
        st["inv_freq"] = _inv_freq(case["rot"], dev) if case["rot"] else None
        if case["mode"] == "accept":
            rng = random.Random(int(seed))
            w = max(1, max(plan["new"]))
            st["picks"] = [sorted(rng.sample(range(case["pack"]), n)) for n in plan["new"]]
            st["keep"] = ints([p + [-1] * (w - len(p)) for p in st["picks"]])
            st["accepted"] = ints(plan["new"])
        elif case["rot"]:
            st["q"] = values(max(total, 1), Hq, D)
            st["q_out"] = torch.zeros_like(st["q"])
        st["cu_q"] = None if case["mode"] == "token" else ints(cu)
        return st
    st["q"] = values(total, Hq, D, scale=1.5)
    st["out"] = torch.empty_like(st["q"])
    if case["op"] == "decode":
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / Hq) for i in range(Hq)], device=dev) if case["alibi"] else None
        st["lse"] = torch.empty((B, Hq), device=dev) if case["lse"] else None
        if own:
            import cast_b200
            n = cast_b200.decode_workspace_size(dtype, B, Hq, Hkv, D)
            st["workspace"] = torch.empty(n, dtype=torch.uint8, device=dev)
        return st
    st["k"], st["v"] = values(total, Hkv, D), values(total, Hkv, D)
    st["cu_q"], st["packs"] = ints(cu), ints(plan["rows"])
    st["parent"] = ints(sum(plan["parents"], []))
    st["words"] = None
    if case["words"]:
        words = []
        for par in plan["parents"]:
            for i, p in enumerate(par):
                words.append((words[len(words) - i + p] if p >= 0 else 0) | (1 << i))
        st["words"] = torch.tensor([w - (1 << 64) if w >= 1 << 63 else w for w in words], dtype=torch.int64, device=dev)
    st["max_pack"], st["max_prefix"] = max(plan["rows"]), max(plan["lens"])
    return st


# ------------------------------------------------------------------------------------------------------ run
def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "tree": _own_tree}[op](state)
    return {"append": _plain_append, "decode": _plain_decode, "tree": _plain_tree}[op](state)


def _own_append(st):
    import cast_b200
    c = st["case"]
    if c["mode"] == "accept":
        cast_b200.append_paged(st["k_pages"], st["v_pages"], st["table"], st["lens"], st["k"], st["v"], st["cu_q"],
                               keep=st["keep"], accepted=st["accepted"], inv_freq=st["inv_freq"],
                               interleaved=c["interleaved"])
        return st["k_pages"], st["v_pages"]
    q = cast_b200.append_paged(st["k_pages"][0], st["v_pages"][0], st["table"], st["lens"], st["k"][0], st["v"][0],
                               st["cu_q"], inv_freq=st["inv_freq"], interleaved=c["interleaved"], q=st.get("q"),
                               q_out=st.get("q_out"))
    return st["k_pages"], st["v_pages"], q


def _own_decode(st):
    import cast_b200
    c = st["case"]
    out = cast_b200.decode_attention_paged(st["q"], st["k_pages"][0], st["v_pages"][0], st["table"], st["lens"],
                                           softcap=c["cap"], window=c["window"], alibi_slopes=st["slopes"],
                                           out=st["out"], lse=st["lse"], workspace=st["workspace"])
    return out, st["lse"]


def _own_tree(st):
    import cast_b200
    words = st["words"]
    return cast_b200.varlen_tree_attention_paged(st["q"], st["k_pages"][0], st["v_pages"][0], st["table"], st["k"],
                                                 st["v"], st["cu_q"], st["lens"], st["packs"], words,
                                                 parent=st["parent"] if words is None else None,
                                                 max_pack=st["max_pack"], max_prefix=st["max_prefix"], out=st["out"])


def _rotate(x, pos, inv_freq, interleaved):
    """x [rows, heads, D] in 32 bits, its first 2 * len(inv_freq) values turned by the angles pos * inv_freq."""
    h = inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq.double()
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    ra, rb = a * c - b * s, b * c + a * s
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., 2 * h:]), -1)


def _plain_append(st):
    c, plan = st["case"], st["plan"]
    dev, ps = st["lens"].device, c["page"]
    total = sum(plan["new"])
    n = torch.tensor(plan["new"], device=dev)
    first = torch.cumsum(n, 0) - n
    seq = torch.repeat_interleave(torch.arange(c["B"], device=dev), n, output_size=total)
    j = torch.arange(total, device=dev) - first[seq]
    slot = st["lens"].long()[seq] + j
    page = st["table"][seq, slot // ps].long()
    row = st["cu_q"].long()[seq] + st["keep"].long()[seq, j] if c["mode"] == "accept" else torch.arange(total, device=dev)
    for kp, vp, k, v in zip(st["k_pages"], st["v_pages"], st["k"], st["v"]):
        new = k[row]
        if c["rot"]:
            new = _rotate(new.float(), slot, st["inv_freq"], c["interleaved"]).to(k.dtype)
        kp[page, :, slot % ps] = new
        vp[page, :, slot % ps] = v[row]
    if c["mode"] == "accept":
        return st["k_pages"], st["v_pages"]
    if c["rot"]:
        q = st["q"][:total]
        st["q_out"][:total] = _rotate(q.float(), slot, st["inv_freq"], c["interleaved"]).to(q.dtype)
    return st["k_pages"], st["v_pages"], st.get("q_out")


def _prefix(pages, table, b, lo, hi, ps):
    """Keys lo..hi-1 of sequence b, [heads, hi - lo, D] in 32 bits."""
    p0, p1 = lo // ps, -(-hi // ps)
    x = pages[table[b, p0:p1].long()].transpose(0, 1).flatten(1, 2)
    return x[:, lo - p0 * ps:hi - p0 * ps].float()


def _plain_decode(st):
    c, ps = st["case"], st["case"]["page"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    for b, n in enumerate(st["plan"]["lens"]):
        lo = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            st["out"][b] = 0
            if c["lse"]:
                st["lse"][b] = -math.inf
            continue
        k = _prefix(st["k_pages"][0], st["table"], b, lo, n, ps)
        v = _prefix(st["v_pages"][0], st["table"], b, lo, n, ps)
        s = torch.matmul(st["q"][b].float().view(Hkv, Hq // Hkv, D), k.transpose(1, 2)) * (1.0 / math.sqrt(D))
        if c["cap"]:
            s = c["cap"] * torch.tanh(s / c["cap"])
        if c["alibi"]:
            s = s + st["slopes"].view(Hkv, -1, 1) * (torch.arange(lo, n, device=s.device) - (n - 1))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        tot = p.sum(-1, keepdim=True)
        st["out"][b] = (torch.matmul(p, v) / tot).reshape(Hq, D).to(st["out"].dtype)
        if c["lse"]:
            st["lse"][b] = (top + torch.log(tot)).reshape(Hq)
    return st["out"], st["lse"]


def _plain_tree(st):
    c, ps, cu = st["case"], st["case"]["page"], st["cu"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    dev = st["q"].device
    for b, (S, P) in enumerate(zip(st["plan"]["lens"], st["plan"]["rows"])):
        rows = slice(cu[b], cu[b + 1])
        k, v = (torch.cat((_prefix(pg, st["table"], b, 0, S, ps), pk[rows].transpose(0, 1).float()), 1)
                for pg, pk in ((st["k_pages"][0], st["k"]), (st["v_pages"][0], st["v"])))
        if st["words"] is not None:
            seen = ((st["words"][rows, None] >> torch.arange(P, device=dev)) & 1).bool()
        else:
            par = st["parent"][rows].long()
            step = torch.zeros(P, P + 1, device=dev)
            step.scatter_(1, torch.where(par < 0, P, par)[:, None], 1.0)
            reach = step[:, :P] + torch.eye(P, device=dev)
            for _ in range(max(1, (P - 1).bit_length())):
                reach = (torch.matmul(reach, reach) > 0).float()
            seen = reach > 0
        q = st["q"][rows].float().view(P, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
        s = (torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(D))).view(Hkv, Hq // Hkv, P, S + P)
        s[..., S:] = s[..., S:].masked_fill(~seen, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p.view(Hkv, -1, S + P), v) / p.view(Hkv, -1, S + P).sum(-1, keepdim=True)
        st["out"][rows] = o.view(Hkv, -1, P, D).permute(2, 0, 1, 3).reshape(P, Hq, D).to(st["out"].dtype)
    return st["out"]


# ---------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "tree": _exact_tree}[case["op"]](st)


def _exact_turn(x, pos, freq, interleaved):
    """One row [heads, D] in 64 bits, pair by pair as a complex number times exp(i pos freq)."""
    h = len(freq)
    turn = np.exp(1j * float(pos) * freq)
    y = x.copy()
    ia, ib = (np.arange(0, 2 * h, 2), np.arange(1, 2 * h, 2)) if interleaved else (np.arange(h), np.arange(h) + h)
    z = (x[:, ia] + 1j * x[:, ib]) * turn
    y[:, ia], y[:, ib] = z.real, z.imag
    return y


def _exact_append(st):
    c, plan, cu = st["case"], st["plan"], st["cu"]
    table = st["table"].cpu().numpy()
    freq = st["inv_freq"].cpu().numpy().astype(np.float64) if c["rot"] else None
    where, src, pos = [], [], []
    for b, n in enumerate(plan["new"]):
        for j in range(n):
            at = plan["lens"][b] + j
            where.append((table[b, at // c["page"]], at % c["page"]))
            src.append(cu[b] + (st["picks"][b][j] if c["mode"] == "accept" else j))
            pos.append(at)
    dev = st["lens"].device
    pg = torch.tensor([w[0] for w in where], dtype=torch.long, device=dev)
    off = torch.tensor([w[1] for w in where], dtype=torch.long, device=dev)

    def turned(x):
        y = x.double()[torch.tensor(src, dtype=torch.long, device=dev)].cpu().numpy()
        if freq is not None:
            for i in range(len(src)):
                y[i] = _exact_turn(y[i], pos[i], freq, c["interleaved"])
        return torch.from_numpy(y).to(dev)

    ks, vs = [], []
    for kp, vp, k, v in zip(st["k_pages"], st["v_pages"], st["k"], st["v"]):
        kp, vp = kp.double(), vp.double()
        if src:
            kp[pg, :, off] = turned(k)
            vp[pg, :, off] = v.double()[torch.tensor(src, dtype=torch.long, device=dev)]
        ks.append(kp)
        vs.append(vp)
    if c["mode"] == "accept":
        return ks, vs
    if not c["rot"]:
        return ks, vs, None
    q = st["q_out"].double()
    q[:len(src)] = turned(st["q"])
    return ks, vs, q


def _exact_rows(pages, table, b, lo, hi, ps):
    at = torch.arange(lo, hi, device=pages.device)
    return pages[table[b].long()[at // ps], :, at % ps].double()      # [keys, heads, D]


def _exact_decode(st):
    c = st["case"]
    Hq, G = c["Hq"], c["Hq"] // c["Hkv"]
    out = torch.zeros((c["B"], Hq, c["D"]), dtype=torch.float64, device=st["q"].device)
    lse = torch.full((c["B"], Hq), -math.inf, dtype=torch.float64, device=out.device)
    for b, n in enumerate(st["plan"]["lens"]):
        lo = n - min(n, c["window"]) if c["window"] else 0
        if n == 0:
            continue
        k = _exact_rows(st["k_pages"][0], st["table"], b, lo, n, c["page"])
        v = _exact_rows(st["v_pages"][0], st["table"], b, lo, n, c["page"])
        for h in range(Hq):
            s = k[:, h // G] @ st["q"][b, h].double() / math.sqrt(c["D"])
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            if c["alibi"]:
                s = s - st["slopes"][h].double() * torch.arange(n - 1 - lo, -1, -1, device=s.device)
            lse[b, h] = torch.logsumexp(s, 0)
            out[b, h] = torch.exp(s - lse[b, h]) @ v[:, h // G]
    return out, lse if c["lse"] else None


def _exact_tree(st):
    c, cu = st["case"], st["cu"]
    Hq, G = c["Hq"], c["Hq"] // c["Hkv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    for b, (S, P) in enumerate(zip(st["plan"]["lens"], st["plan"]["rows"])):
        rows = slice(cu[b], cu[b + 1])
        k = torch.cat((_exact_rows(st["k_pages"][0], st["table"], b, 0, S, c["page"]), st["k"][rows].double()))
        v = torch.cat((_exact_rows(st["v_pages"][0], st["table"], b, 0, S, c["page"]), st["v"][rows].double()))
        hide = np.zeros((P, S + P), dtype=bool)
        hide[:, S:] = True
        for i in range(P):
            a = i
            while a >= 0:
                hide[i, S + a] = False
                a = st["plan"]["parents"][b][a]
        hide = torch.from_numpy(hide).to(out.device)
        for h in range(Hq):
            s = (st["q"][rows, h].double() @ k[:, h // G].T / math.sqrt(c["D"])).masked_fill(hide, -math.inf)
            out[rows, h] = torch.softmax(s, -1) @ v[:, h // G]
    return out
