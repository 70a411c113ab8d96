"""The operators that take a decode session from one greedy answer to several drawn ones, and the cases they are timed on.

sample   one token a row from logits: temperature, top-k, top-p and min-p, drawn with a random number that is given
pages    pages of the paged KV cache: copied between pools, shared by forked sequences, moved together, given back
attn     one layer's decode attention for sequences that share a long prefix, whose keys and values are read once for all of them

`run` computes them from elementary torch operations where `own` is false, and calls the framework where it is true.
"""
import math
import random

import torch

import etx_megakernel_b200  # noqa: F401  (registers the package)

own = False
DEV = 0
PAGE = 16                                                               # positions of a page


def listed():
    return [
        # ---- sample
        # the token of one conversation, vocabulary and settings of a chat model: latency is all there is
        {"name": "sample-1x151936", "kind": "sample", "rows": 1, "V": 151936, "dtype": "bf16", "set": "chat", "masked": 0.0},
        # a batch of the benchmark's size, every request with settings of its own, a part of them greedy
        {"name": "sample-32x151936-mixed", "kind": "sample", "rows": 32, "V": 151936, "dtype": "bf16", "set": "mixed", "masked": 0.0},
        # logits that a user's program corrected in fp32, most of the vocabulary forbidden by a grammar; no size is round
        {"name": "sample-13x50257-f32", "kind": "sample", "rows": 13, "V": 50257, "dtype": "f32", "set": "mixed", "masked": 0.7},
        # rollouts: many answers at temperature 1 with nothing cut off, where the whole vocabulary counts
        {"name": "sample-256x151936-open", "kind": "sample", "rows": 256, "V": 151936, "dtype": "bf16", "set": "open", "masked": 0.0},
        # ---- pages
        # one prompt of 1037 positions becomes eight answers: full pages shared, the last one copied, tables written
        {"name": "pages-fork-8", "kind": "fork", "layers": 48, "nkv": 4, "hd": 128, "length": 1037, "forks": 8},
        # a prompt computed by a one-sequence session moves into the pool of a batch
        {"name": "pages-copy-257", "kind": "copy", "layers": 24, "nkv": 8, "hd": 128, "pages": 257},
        # the life of a pool: forked, grown, every second answer ends, the rest moved together, all given back
        {"name": "pages-life-32", "kind": "life", "layers": 12, "nkv": 4, "hd": 128, "length": 515, "forks": 32, "grow": 90},
        # ---- attn
        # a few answers to a short prompt
        {"name": "attn-4seq-1k", "kind": "attn", "nh": 32, "nkv": 4, "hd": 128, "seqs": 4, "groups": 1, "prefix": 1024, "own": 33, "ragged": False},
        # the benchmark's batch over a document of 8000 positions, answers of different lengths
        {"name": "attn-32seq-8k", "kind": "attn", "nh": 32, "nkv": 4, "hd": 128, "seqs": 32, "groups": 1, "prefix": 8150, "own": 300, "ragged": True},
        # several prompts, each with answers of its own, six query heads for a kv head: nothing is a multiple of anything
        {"name": "attn-21seq-5groups", "kind": "attn", "nh": 12, "nkv": 2, "hd": 128, "seqs": 21, "groups": 5, "prefix": 2003, "own": 77, "ragged": True},
        # two answers over a very long context
        {"name": "attn-2seq-128k", "kind": "attn", "nh": 32, "nkv": 8, "hd": 128, "seqs": 2, "groups": 1, "prefix": 131000, "own": 1000, "ragged": True},
        # a wide batch over a long context: the shared part is a matrix product with hundreds of rows
        {"name": "attn-64seq-32k", "kind": "attn", "nh": 32, "nkv": 8, "hd": 128, "seqs": 64, "groups": 1, "prefix": 32500, "own": 500, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["sample", "sample", "attn", "attn", "attn", "fork", "copy", "life"])
    if kind == "sample":
        V = _log_int(rng, 300, 262144)
        return {"kind": kind, "rows": min(_log_int(rng, 1, 256), 128 * 151936 // V), "V": V, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "set": rng.choice(["chat", "mixed", "mixed", "open"]), "masked": rng.choice([0.0, 0.0, 0.3, 0.9])}
    if kind == "attn":
        nkv, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 6, 8])
        seqs = _log_int(rng, 1, 96)
        c = {"kind": kind, "nh": nkv * G, "nkv": nkv, "hd": rng.choice([64, 80, 128, 128, 256]), "seqs": seqs, "groups": min(seqs, rng.choice([1, 1, 2, 3, 7])),
             "prefix": _log_int(rng, 5, 65536), "own": _log_int(rng, 1, 1500), "ragged": rng.choice([True, True, False])}
        top = work(listed()[-1])
        while work(c)["flops"] > top["flops"] or work(c)["bytes"] > top["bytes"]:
            c["prefix"], c["own"] = c["prefix"] * 3 // 4 + 1, c["own"] * 3 // 4 + 1
        return c
    layers, nkv, hd = _log_int(rng, 1, 48), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    page = 2 * 2 * PAGE * nkv * hd * layers                              # bytes of one page, keys and values of all layers
    if kind == "copy":
        return {"kind": kind, "layers": layers, "nkv": nkv, "hd": hd, "pages": max(1, min(_log_int(rng, 1, 600), 400_000_000 // page))}
    c = {"kind": kind, "layers": layers, "nkv": nkv, "hd": hd, "length": _log_int(rng, 1, 4000), "forks": _log_int(rng, 1, 48)}
    if kind == "life":
        c["grow"] = _log_int(rng, 1, 200)
        while (c["length"] // PAGE + 2 + c["forks"] * (2 + c["grow"] // PAGE)) * page > 1_500_000_000:
            c["length"], c["forks"], c["grow"] = c["length"] * 2 // 3 + 1, max(1, c["forks"] * 2 // 3), c["grow"] * 2 // 3 + 1
    else:
        while (c["length"] // PAGE + 2 + c["forks"]) * page > 1_500_000_000:
            c["length"], c["forks"] = c["length"] * 2 // 3 + 1, max(1, c["forks"] * 2 // 3)
    return c


# ------------------------------------------------------------------------------------------------ shapes that follow from a case
def _lens(case):
    """(sequences of each group, prefix length of each group, own length of each sequence)."""
    rng = random.Random(case["seqs"] * 1000003 + case["prefix"] * 101 + case["own"])
    n, g = case["seqs"], case["groups"]
    sizes = [n // g + (1 if i < n % g else 0) for i in range(g)]
    if case["ragged"] and g > 1:
        for i in range(0, g - 1, 2):                                    # uneven groups
            k = rng.randint(0, sizes[i] - 1)
            sizes[i] -= k
            sizes[i + 1] += k
    if not case["ragged"]:
        return sizes, [case["prefix"]] * g, [case["own"]] * n
    return sizes, [max(1, case["prefix"] - rng.randint(0, case["prefix"] // 3) * (i > 0)) for i in range(g)], [rng.randint(1, case["own"]) for _ in range(n)]


def _np(n):
    return -(-n // PAGE)


def _pool_pages(case):
    if case["kind"] == "fork":
        return _np(case["length"]) + case["forks"] + 3
    return _np(case["length"]) + case["forks"] * (2 + _np(case["grow"])) + 3


# ------------------------------------------------------------------------------------------------ prepare
def prepare(case, seed):
    dev = torch.device("cuda", DEV)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    state = {"case": dict(case)}
    return {"sample": _prepare_sample, "fork": _prepare_pool, "life": _prepare_pool, "copy": _prepare_copy, "attn": _prepare_attn}[case["kind"]](case, state, dev, gen, seed)


def _prepare_sample(case, s, dev, gen, seed):
    B, V = case["rows"], case["V"]
    # scores like a language model's: a broad bell, and a tail of a few likely tokens
    l = torch.empty((B, V), device=dev).normal_(0.0, 2.0, generator=gen)
    top = torch.empty((B, 40), device=dev).exponential_(1.0, generator=gen) * 2.0 + 8.0
    l.scatter_(1, torch.randint(0, V // 40, top.shape, device=dev, generator=gen) + torch.arange(40, device=dev) * (V // 40), top)
    if case["masked"]:
        l.masked_fill_(torch.rand((B, V), device=dev, generator=gen) < case["masked"], float("-inf"))
        l[:, 0].clamp_(min=-3.0)                                        # the end of the answer stays allowed
    s["logits"] = l.to({"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]])
    s["u"] = torch.rand(B, device=dev, generator=gen)
    rng = random.Random(seed)
    if case["set"] == "chat":
        rows = [(0.7, 50, 0.9, 0.0)] * B
    elif case["set"] == "open":
        rows = [(1.0, 0, 1.0, 0.0)] * B
    else:
        rows = [rng.choice([(0.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 0, 0.95, 0.0), (1.3, 0, 1.0, 0.05), (0.9, 200, 0.97, 0.01), (1.0, 0, 1.0, 0.0)]) for _ in range(B)]
    s["temperature"] = torch.tensor([r[0] for r in rows], device=dev)
    s["top_k"] = torch.tensor([r[1] for r in rows], dtype=torch.int32, device=dev)
    s["top_p"] = torch.tensor([r[2] for r in rows], device=dev)
    s["min_p"] = torch.tensor([r[3] for r in rows], device=dev)
    return s


def _cache(case, pages, dev, gen):
    """Keys and values of all layers in the paged layout, random everywhere."""
    k = torch.empty((case["layers"], pages, case["nkv"], case["hd"] // 8, PAGE, 8), dtype=torch.bfloat16, device=dev).normal_(0.0, 1.0, generator=gen)
    v = torch.empty((case["layers"], pages, case["nkv"], case["hd"], PAGE), dtype=torch.bfloat16, device=dev).normal_(0.0, 0.9, generator=gen)
    return k, v


def _prepare_pool(case, s, dev, gen, seed):
    pages = _pool_pages(case)
    s["kc"], s["vc"] = _cache(case, pages, dev, gen)
    width = _np(case["length"] + case.get("grow", 0)) + 1
    if own:
        from etx_megakernel_b200.runtime import PagePool
        s["pool"] = PagePool([s["kc"], s["vc"]], max_seqs=case["forks"] + 1, max_pages=width)
        s["row"] = s["pool"].open(case["length"])
    else:
        s["tables"] = torch.zeros((case["forks"] + 1, width), dtype=torch.int32, device=dev)
        n = _np(case["length"])
        s["tables"][0, :n] = torch.arange(n, dtype=torch.int32, device=dev)
        s["held"] = list(range(n))                                       # the prompt's pages
    return s


def _prepare_copy(case, s, dev, gen, seed):
    n = case["pages"]
    s["src"] = _cache(case, n + 2, dev, gen)
    s["dst"] = _cache(case, n + 9, dev, gen)
    rng = random.Random(seed)
    s["src_ids"], s["dst_ids"] = rng.sample(range(n + 2), n), rng.sample(range(n + 9), n)
    return s


def _prepare_attn(case, s, dev, gen, seed):
    sizes, plens, lens = _lens(case)
    need = sum(_np(p) for p in plens) + sum(_np(n) for n in lens)
    k, v = _cache(dict(case, layers=1), need + 1, dev, gen)
    s["kc"], s["vc"] = k[0], v[0]
    s["q"] = torch.empty((case["seqs"], case["nh"], case["hd"]), dtype=torch.bfloat16, device=dev).normal_(0.0, 1.3, generator=gen)
    order = torch.randperm(need, device=dev, generator=gen).to(torch.int32)     # the pages of a pool in use lie anywhere
    s["prefix_tables"] = torch.full((case["groups"], max(_np(p) for p in plens)), need, dtype=torch.int32, device=dev)
    s["tables"] = torch.full((case["seqs"], max(_np(n) for n in lens)), need, dtype=torch.int32, device=dev)
    at = 0
    for table, lengths in ((s["prefix_tables"], plens), (s["tables"], lens)):
        for i, n in enumerate(lengths):
            table[i, :_np(n)] = order[at:at + _np(n)]
            at += _np(n)
    s["prefix_lens"] = torch.tensor(plens, dtype=torch.int32, device=dev)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["sizes"], s["host_plens"], s["host_lens"] = sizes, plens, lens
    s["scale"] = case["hd"] ** -0.5
    return s


# ------------------------------------------------------------------------------------------------ run
def run(state):
    return {"sample": _run_sample, "fork": _run_fork, "life": _run_life, "copy": _run_copy, "attn": _run_attn}[state["case"]["kind"]](state)


def _run_sample(s):
    if own:
        from etx_megakernel_b200.runtime import sample
        r = sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": r.tokens, "logprobs": r.logprobs, "kept": r.kept}
    # tokens in the order of their scores, equal ones by their index; all three cuts keep a beginning of that order
    l = s["logits"].float()
    l = torch.where(torch.isnan(l), torch.full_like(l, float("-inf")), l)
    order, index = torch.sort(l, dim=1, descending=True, stable=True)
    live = order > float("-inf")
    T = s["temperature"].double()[:, None]
    greedy = ~(T > 0)
    z = (order.double() - order[:, :1].double()) / torch.where(greedy, torch.ones_like(T), T)
    z = torch.where(order == order[:, :1], torch.zeros_like(z), z)
    w = torch.where(live, torch.exp(z), torch.zeros_like(z))
    cum = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
    at = torch.arange(l.shape[1], device=l.device)[None]
    n_live = live.sum(1, keepdim=True)
    k = s["top_k"].long()[:, None]
    nk = torch.where(k > 0, torch.minimum(k, n_live), n_live)
    Wk = cum.gather(1, (nk - 1).clamp(min=0))
    p = s["top_p"].double()[:, None]
    keep = (at < nk) & ((before < p * Wk) | ~(p < 1)) & ((w >= s["min_p"].double()[:, None]) | ~(s["min_p"][:, None] > 0))
    n = keep.sum(1, keepdim=True).clamp(min=1)
    n = torch.where(greedy, torch.ones_like(n), n)
    Wn = cum.gather(1, n - 1)
    u = s["u"].double().clamp(0.0, 1.0 - 2.0 ** -24)[:, None]
    r = torch.minimum((cum <= u * Wn).sum(1, keepdim=True), n - 1)
    empty = n_live[:, 0] == 0
    logp = (z.gather(1, r) - torch.log(Wn))[:, 0]
    return {"tokens": torch.where(empty, -1, index.gather(1, r)[:, 0]).to(torch.int32),
            "logprobs": torch.where(empty, float("-inf"), logp).float(), "kept": torch.where(empty, 0, n[:, 0]).to(torch.int32)}


def _copy_plain(kc, vc, src, dst):
    if src:
        a, b = torch.tensor(src, device=kc.device), torch.tensor(dst, device=kc.device)
        kc[:, b] = kc[:, a]
        vc[:, b] = vc[:, a]


def _fork_plain(s, free):
    """Shares the prompt's full pages with rows 1 .. forks, copies its last, partly filled one; returns the rows' own pages."""
    c, tab = s["case"], s["tables"]
    full, part = divmod(c["length"], PAGE)
    tab[1:c["forks"] + 1, :full] = tab[:1, :full]
    mine = [[free.pop(0)] if part else [] for _ in range(c["forks"])]
    if part:
        _copy_plain(s["kc"], s["vc"], [s["held"][full]] * c["forks"], [m[0] for m in mine])
        tab[1:c["forks"] + 1, full] = torch.tensor([m[0] for m in mine], dtype=torch.int32, device=tab.device)
    return mine


def _run_fork(s):
    c = s["case"]
    if own:
        rows = s["pool"].fork(s["row"], c["forks"])
        s["pool"].close(rows)
        return {"kc": s["kc"], "vc": s["vc"], "tables": s["pool"].tables}
    held = set(s["held"])
    _fork_plain(s, [i for i in range(s["kc"].shape[1]) if i not in held])
    return {"kc": s["kc"], "vc": s["vc"], "tables": s["tables"]}


def _run_life(s):
    c = s["case"]
    length, F = c["length"], c["forks"]
    if own:
        pool = s["pool"]
        rows = pool.fork(s["row"], F)
        pool.extend(rows, length + c["grow"])
        pool.close(rows[::2])
        pool.compact()
        pool.close(rows[1::2])
        return {"kc": s["kc"], "vc": s["vc"], "tables": pool.tables}
    held, full, tab = set(s["held"]), length // PAGE, s["tables"]
    free = [i for i in range(s["kc"].shape[1]) if i not in held]
    mine = _fork_plain(s, free)
    need = _np(length + c["grow"]) - full
    for i in range(F):                                                   # lowest free pages first, row by row
        while len(mine[i]) < need:
            mine[i].append(free.pop(0))
    if need:
        tab[1:F + 1, full:full + need] = torch.tensor(mine, dtype=torch.int32, device=tab.device)
    left = list(range(1, F, 2))                                          # rows 2, 4, ... of the table go on
    used = sorted(held | {p for i in left for p in mine[i]})
    low = [i for i in range(len(used)) if i not in set(used)]            # holes below, pages above: the highest into the lowest
    high = [p for p in used if p >= len(used)][::-1]
    _copy_plain(s["kc"], s["vc"], high, low)
    to = dict(zip(high, low))
    if left and need:
        tab[torch.tensor(left, device=tab.device) + 1, full:full + need] = torch.tensor([[to.get(p, p) for p in mine[i]] for i in left], dtype=torch.int32, device=tab.device)
    return {"kc": s["kc"], "vc": s["vc"], "tables": tab}


def _run_copy(s):
    if own:
        from etx_megakernel_b200.runtime import copy_pages
        copy_pages(s["src"], s["dst"], s["src_ids"], s["dst_ids"])
    else:
        a, b = torch.tensor(s["src_ids"], device=s["src"][0].device), torch.tensor(s["dst_ids"], device=s["src"][0].device)
        for x, y in zip(s["src"], s["dst"]):
            y[:, b] = x[:, a]
    return {"kc": s["dst"][0], "vc": s["dst"][1]}


def _rows(kc, vc, pages, n, dt):
    """[n][NKV][HD] keys and values of the positions that `pages` hold."""
    p = pages.long()
    k = kc[p].permute(0, 3, 1, 2, 4).reshape(-1, kc.shape[1], kc.shape[2] * kc.shape[4])[:n]
    v = vc[p].permute(0, 3, 1, 2).reshape(-1, vc.shape[1], vc.shape[2])[:n]
    return k.to(dt), v.to(dt)


def _run_attn(s):
    if own:
        from etx_megakernel_b200.runtime import attn_shared
        return {"out": attn_shared(s["q"], s["kc"], s["vc"], s["tables"], s["lens"], s["prefix_tables"], s["prefix_lens"], groups=s["sizes"], scale=s["scale"])}
    nkv, hd = s["kc"].shape[1], s["q"].shape[2]
    G = s["q"].shape[1] // nkv
    q = s["q"].float().view(-1, nkv, G, hd) * s["scale"]
    out = torch.empty_like(s["q"])
    b = 0
    for g, n in enumerate(s["sizes"]):
        pk, pv = _rows(s["kc"], s["vc"], s["prefix_tables"][g, :_np(s["host_plens"][g])], s["host_plens"][g], torch.float32)
        pk, pv = pk.transpose(0, 1), pv.transpose(0, 1)                  # [nkv][positions][hd]
        qg = q[b:b + n].permute(1, 0, 2, 3).reshape(nkv, n * G, hd)
        sp = torch.matmul(qg, pk.transpose(1, 2))                        # the shared part, once for all rows
        m = sp.amax(2, keepdim=True)
        own_scores = []
        for i in range(n):
            ln = s["host_lens"][b + i]
            ok, ov = _rows(s["kc"], s["vc"], s["tables"][b + i, :_np(ln)], ln, torch.float32)
            sc = torch.matmul(qg[:, i * G:(i + 1) * G], ok.permute(1, 2, 0))
            m[:, i * G:(i + 1) * G] = torch.maximum(m[:, i * G:(i + 1) * G], sc.amax(2, keepdim=True))
            own_scores.append((sc, ov))
        e = torch.exp(sp - m)
        num, den = torch.matmul(e, pv), e.sum(2, keepdim=True)
        for i, (sc, ov) in enumerate(own_scores):
            e = torch.exp(sc - m[:, i * G:(i + 1) * G])
            num[:, i * G:(i + 1) * G] += torch.matmul(e, ov.transpose(0, 1))
            den[:, i * G:(i + 1) * G] += e.sum(2, keepdim=True)
        out[b:b + n] = (num / den).view(nkv, n, G, hd).permute(1, 0, 2, 3).reshape(n, nkv * G, hd).to(out.dtype)
        b += n
    return {"out": out}


# ------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """The definitions in 64 bits, written apart from the plain forms."""
    if case["kind"] in ("fork", "life", "copy"):
        return _exact_pages(case, prepare(case, seed))
    s = prepare(case, seed)
    if case["kind"] == "sample":
        tokens, logps, kept = [], [], []
        for b in range(case["rows"]):
            l = s["logits"][b].double()
            T, k, p, mp = (float(s[n][b]) for n in ("temperature", "top_k", "top_p", "min_p"))
            ids = torch.nonzero(l > float("-inf"))[:, 0]
            v, o = torch.sort(l[ids], descending=True, stable=True)
            n = v.numel() if k <= 0 else min(int(k), v.numel())
            if not T > 0:
                n, T = 1, 1.0
            w = torch.exp((v - v[0]) / T)
            c = torch.cumsum(w[:n], 0)
            if p < 1:
                n = min(n, int((c < p * c[-1]).sum()) + 1)              # up to the first that reaches p
            if mp > 0:
                n = min(n, max(1, int((w >= mp).sum())))
            c = c[:n]
            r = min(int(torch.searchsorted(c, float(s["u"][b]) * c[-1], right=True)), n - 1)
            tokens.append(int(ids[o[r]]))
            logps.append(float((v[r] - v[0]) / T - torch.log(c[-1])))
            kept.append(n)
        dev = s["logits"].device
        return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=dev), "logprobs": torch.tensor(logps, dtype=torch.float64, device=dev),
                "kept": torch.tensor(kept, dtype=torch.int32, device=dev)}
    G = case["nh"] // case["nkv"]
    rows, b = [], 0
    for g, n in enumerate(s["sizes"]):
        pk, pv = _rows(s["kc"], s["vc"], s["prefix_tables"][g, :_np(s["host_plens"][g])], s["host_plens"][g], torch.bfloat16)
        for i in range(b, b + n):
            ln = s["host_lens"][i]
            ok, ov = _rows(s["kc"], s["vc"], s["tables"][i, :_np(ln)], ln, torch.bfloat16)
            heads = []
            for h in range(case["nkv"]):                                 # one head at a time: 64-bit copies of a long context are large
                K, V = torch.cat([pk[:, h], ok[:, h]]).double(), torch.cat([pv[:, h], ov[:, h]]).double()
                heads.append(torch.softmax(s["q"][i, h * G:(h + 1) * G].double() @ K.T * s["scale"], dim=1) @ V)
            rows.append(torch.cat(heads))
        b += n
    return {"out": torch.stack(rows)}


def _exact_pages(case, s):
    """Which page of the beginning every page holds at the end, followed page by page; the tables likewise."""
    if case["kind"] == "copy":
        out = [y.double() for y in s["dst"]]
        for a, b in zip(s["src_ids"], s["dst_ids"]):
            for x, y in zip(s["src"], out):
                y[:, b] = x[:, a].double()
        return {"kc": out[0], "vc": out[1]}
    length, F, total = case["length"], case["forks"], s["kc"].shape[1]
    holds = list(range(total))
    seq = {0: list(range(_np(length)))}                                  # pages of each sequence, in order
    users = {p: 1 for p in seq[0]}

    def take():
        p = min(i for i in range(total) if i not in users)
        users[p] = 1
        return p
    for f in range(1, F + 1):
        seq[f] = seq[0][:length // PAGE]
        for p in seq[f]:
            users[p] += 1
    if length % PAGE:
        for f in range(1, F + 1):
            seq[f].append(take())
            holds[seq[f][-1]] = holds[seq[0][-1]]
    shown = {f: list(t) for f, t in seq.items()}                         # what the tables show
    if case["kind"] == "life":
        for f in range(1, F + 1):
            while len(seq[f]) * PAGE < length + case["grow"]:
                seq[f].append(take())
            shown[f] = list(seq[f])
        for f in range(1, F + 1, 2):
            for p in seq.pop(f):
                users[p] -= 1
                if not users[p]:
                    del users[p]
        while True:
            top, hole = max(users), min(i for i in range(total + 1) if i not in users)
            if hole > top:
                break
            holds[hole] = holds[top]
            users[hole] = users.pop(top)
            for f, t in seq.items():
                seq[f] = [hole if p == top else p for p in t]
                shown[f] = list(seq[f])
    width = _np(length + case.get("grow", 0)) + 1
    tables = torch.zeros((F + 1, width), dtype=torch.int32)
    for f, t in shown.items():
        tables[f, :len(t)] = torch.tensor(t, dtype=torch.int32)
    at = torch.tensor(holds, device=s["kc"].device)
    return {"kc": s["kc"][:, at].double(), "vc": s["vc"][:, at].double(), "tables": tables.to(s["kc"].device)}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "sample":
        size = 4 if case["dtype"] == "f32" else 2
        n = case["rows"] * case["V"]
        return {"bytes": n * size + case["rows"] * 32, "flops": 2.0 * n}           # a weight and its sum
    if kind == "attn":
        sizes, plens, lens = _lens(case)
        G = case["nh"] // case["nkv"]
        row = 2 * 2 * case["nkv"] * case["hd"]                                     # a position's key and value
        kv = sum(plens) + sum(lens)
        pairs = sum(n * p for n, p in zip(sizes, plens)) + sum(lens)
        return {"bytes": row * kv + 2 * 2 * case["seqs"] * case["nh"] * case["hd"], "flops": 4.0 * case["nkv"] * G * case["hd"] * pairs}
    page = 2 * 2 * PAGE * case["nkv"] * case["hd"] * case["layers"]
    if kind == "copy":
        return {"bytes": 2 * case["pages"] * page, "flops": 0.0}
    full, part = divmod(case["length"], PAGE)
    tables = 4 * case["forks"] * (full + 1)
    if kind == "fork":
        return {"bytes": (1 + case["forks"]) * page * (part > 0) + 2 * tables, "flops": 0.0}
    need = _np(case["length"] + case["grow"]) - full
    held, F = _np(case["length"]), case["forks"]
    n_used = held + (F // 2) * need                                                # every second answer's pages, moved below this line
    pages = _life_pages(case)
    moved = sum(1 for i in range(1, F, 2) for p in pages[i] if p >= n_used)
    return {"bytes": (1 + F) * page * (part > 0) + 2 * moved * page + 3 * tables, "flops": 0.0}


def _life_pages(case):
    """The pages that the forks of a `life` case hold once they have grown: the lowest free ones, row by row."""
    full, part = divmod(case["length"], PAGE)
    need, at = _np(case["length"] + case["grow"]) - full, _np(case["length"])
    mine = [[] for _ in range(case["forks"])]
    if part:
        for m in mine:
            m.append(at)
            at += 1
    for m in mine:
        while len(m) < need:
            m.append(at)
            at += 1
    return mine
