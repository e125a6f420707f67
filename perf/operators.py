"""The serving operators of First Passage Attention, as measured cases: a paged cache that is quantised as it is
written and read back, the attention of the newest tokens over it (with or without a prefix that the whole batch
shares), and the verification of drafted tokens.

Every case is real work of a language model that answers: sizes follow the language model (12 heads of 64, 50304
tokens in the vocabulary, contexts of 2048) and the operator benchmarks (8 heads, T 1000, head dimensions 16 to 256;
16 heads of 128, T 16383).

``run`` computes an operator in its plain form (elementary torch operations in float32) or, with ``own`` set,
through the package's public entry points. ``exact`` computes the same in float64 from the definitions.
"""
import math
import random

import torch

own = False

PAGE = 64
DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------- cases ----

def listed():
    return [
        # One step of a batch of 32 requests: each writes the token it has just computed into its int8 cache, and
        # reads it back as attention would see it.
        dict(name="append_step", kind="append", B=32, H=12, D=64, L=2048, n=1, type="fp16", int8=True, mix=1, page=64),
        # Four prompts of the language model's context length enter an int8 cache.
        dict(name="append_prompts", kind="append", B=4, H=12, D=64, L=2048, n=2048, type="fp16", int8=True, mix=2,
             page=64),
        # Odd chunks of prompts in float32 into an unquantised cache that they do not start at a page of.
        dict(name="append_fp32", kind="append", B=3, H=8, D=32, L=1000, n=333, type="fp32", int8=False, mix=3, page=32),
        # The whole histories of eight long requests, taken out of the int8 cache (to move or to re-prefill them).
        dict(name="read_long", kind="read", B=8, H=16, D=128, L=16383, n=16383, type="fp16", int8=True, mix=4,
             page=128),
        # A single request, one token: nothing but latency.
        dict(name="decode_one", kind="decode", B=1, H=12, D=64, L=1000, n=1, P=0, type="fp16", int8=False, mix=5,
             page=64),
        # A batch of 64 requests at mixed lengths, one token each, int8 cache: the ordinary serving step.
        dict(name="decode_batch", kind="decode", B=64, H=12, D=64, L=2048, n=1, P=0, type="fp16", int8=True, mix=6,
             page=64),
        # Four long contexts with five drafted tokens to check, fp16 cache, the benchmark's 16 heads of 128.
        dict(name="decode_long_draft", kind="decode", B=4, H=16, D=128, L=16383, n=5, P=0, type="fp16", int8=False,
             mix=7, page=128),
        # The float32 model: three tokens a step, odd length.
        dict(name="decode_fp32", kind="decode", B=8, H=8, D=32, L=1000, n=3, P=0, type="fp32", int8=False, mix=8,
             page=32),
        # 64 requests behind one system prompt of 8192 tokens, own parts of up to 512, int8 cache.
        dict(name="prefix_batch", kind="decode", B=64, H=12, D=64, L=512, n=1, P=8192, type="fp16", int8=True, mix=9,
             page=64),
        # 24 samples of one question behind a document of 16383 tokens, five drafted tokens each, fp16 cache.
        dict(name="prefix_draft", kind="decode", B=24, H=16, D=128, L=1000, n=5, P=16383, type="fp16", int8=False,
             mix=10, page=128),
        # One request with four drafted tokens, the language model's vocabulary.
        dict(name="verify_one", kind="verify", B=1, n=4, V=50304, type="fp32", mix=11),
        # A batch of 64 requests with seven drafted tokens each.
        dict(name="verify_batch", kind="verify", B=64, n=7, V=50304, type="fp32", mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: batches of 1 to 64 (256 for the verification), 1 to 16 heads, every head dimension,
    contexts of 1 to 16383 tokens, 1 to 16 new tokens, prefixes up to 16383, both types, int8 or not."""
    while True:
        kind = rng.choice(["append", "read", "decode", "decode", "prefix", "prefix", "verify"])
        mix, typ = rng.randrange(1 << 20), rng.choice(["fp16", "fp16", "fp32"])
        if kind == "verify":
            c = dict(kind="verify", B=_log(rng, 1, 256), n=rng.randint(1, 16), V=_log(rng, 1000, 50304), type=typ,
                     mix=mix)
        else:
            c = dict(kind="decode" if kind == "prefix" else kind, B=_log(rng, 1, 64), H=rng.randint(1, 16),
                     D=rng.choice([16, 32, 64, 64, 128, 128, 256]), type=typ, int8=rng.random() < 0.6, mix=mix,
                     page=rng.choice([32, 64, 128, 256]))
            c["L"] = _log(rng, 1, 2048 if kind == "prefix" else 16383)
            if kind in ("append", "read"):
                c["n"] = min(c["L"], _log(rng, 1, 16383))
            else:
                c["n"] = min(c["L"], rng.choice([1, 1, rng.randint(2, 16)]))
                c["P"] = _log(rng, 64, 16383) if kind == "prefix" else 0
        w = work(c)
        # No more than the largest listed cases: in bytes (also of the plain form's float32 copies) and in products.
        size = c["B"] * c.get("H", 1) * c.get("D", 1) * (c.get("L", 0) + c.get("P", 0))
        flops = 4e9 if c["type"] == "fp32" else 1.6e10
        if w["bytes"] <= 6e8 and w["flops"] <= flops and size <= 2.5e8:
            return c


def _lens(case):
    """Tokens of each sequence, the newest ones included: the first has L, the others between L/4 and L; in batches
    of more than eight one slot is idle (0 tokens)."""
    rng = random.Random(case["mix"])
    L = case["L"]
    lens = [L] + [rng.randint(max(1, L // 4), L) for _ in range(case["B"] - 1)]
    if case["kind"] == "decode" and case["B"] > 8:
        lens[rng.randrange(1, case["B"])] = 0
    return lens


def _counts(case):
    """Tokens that each sequence appends or has read: its last n, or all that it has."""
    return [min(case["n"], x) for x in _lens(case)]


# ------------------------------------------------------------------------------------------------------ inputs ----

def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _field(g, *shape):
    """phi and psi of a trained field's scale: a walk with steps of a half, offsets of one."""
    walk = (0.5 * torch.randn(*shape, generator=g, device=DEVICE)).cumsum(-1)
    return (walk + torch.randn(*shape, generator=g, device=DEVICE),
            walk + torch.randn(*shape, generator=g, device=DEVICE))


def _kv(g, case, B, T):
    """Keys and values with channels of unlike size, as projections give them."""
    out = []
    for _ in range(2):
        gain = torch.exp(0.5 * torch.randn(case["H"], 1, case["D"], generator=g, device=DEVICE))
        x = torch.randn(B, case["H"], T, case["D"], generator=g, device=DEVICE)
        out.append(x.mul_(gain).to(DTYPES[case["type"]]))
    return out


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def _tables(case, g):
    """Pages in no order, a table row for each sequence (unused entries -1) and the prefix's table."""
    page = case["page"]
    need = [-(-x // page) for x in _lens(case)]
    npre = -(-case.get("P", 0) // page)
    n_pages = sum(need) + npre + 3
    perm = torch.randperm(n_pages, generator=g, device=DEVICE).tolist()
    width = max(need)
    rows, at = [], 0
    for x in need:
        rows.append(perm[at:at + x] + [-1] * (width - x))
        at += x
    return n_pages, _int32(rows), _int32(perm[at:at + npre])


def _sequences(case, seed):
    """Everything random of a cache case, in one order: tables, own keys, values and field, the prefix's, queries."""
    g = _gen(seed)
    B, H, D = case["B"], case["H"], case["D"]
    n_pages, table, ptable = _tables(case, g)
    d = dict(n_pages=n_pages, table=table, ptable=ptable)
    d["k"], d["v"] = _kv(g, case, B, case["L"])
    d["phi"], d["psi"] = _field(g, B, H, case["L"])
    if case.get("P"):
        d["pk"], d["pv"] = _kv(g, case, 1, case["P"])
        d["pphi"], d["ppsi"] = _field(g, 1, H, case["P"])
        d["phi"] += d["pphi"][..., -1:]  # the walk goes on where the prefix's ends
        d["psi"] += d["pphi"][..., -1:]
    if case["kind"] == "decode":
        d["q"] = torch.randn(B, H, case["n"], D, generator=g, device=DEVICE).to(DTYPES[case["type"]])
        d["beta"] = 0.5 + torch.rand(H, generator=g, device=DEVICE)
    return d


def _quantise(x):
    """int8 codes and a scale for each row, in float32: scale = max|x| / 127, code = rint(127 x / max|x|)."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    top = torch.where(top == 0, torch.full_like(top, 127.0), top)
    return torch.round((x * 127.0) / top).to(torch.int8), (top / 127.0).squeeze(-1)


def _plain_pool(case, n_pages):
    """The plain form's paged pool, entries [pages, heads, page, ...], with a spare page at its end."""
    H, D, page = case["H"], case["D"], case["page"]
    dt = torch.int8 if case["int8"] else DTYPES[case["type"]]
    pool = {n: torch.zeros(n_pages + 1, H, page, D, dtype=dt, device=DEVICE) for n in "kv"}
    for n in ("phi", "psi") + (("ks", "vs") if case["int8"] else ()):
        pool[n] = torch.zeros(n_pages + 1, H, page, device=DEVICE)
    return pool


def _plain_write(pool, table, start, count, k, v, phi, psi):
    """Writes count_b tokens of each sequence at its positions start_b on; the others go to the last, spare page."""
    page = pool["k"].shape[2]
    i = torch.arange(k.shape[2], device=DEVICE)
    pos = start[:, None].long() + i
    pid = table.long().gather(1, (pos // page).clamp(max=table.shape[1] - 1))
    pid = torch.where(i < count[:, None], pid, pool["k"].shape[0] - 1)
    off = pos % page
    for name, x in (("k", k), ("v", v)):
        rows = x.permute(0, 2, 1, 3)
        if pool["k"].dtype == torch.int8:
            codes, scale = _quantise(rows)
            pool[name][pid, :, off] = codes
            pool[name + "s"][pid, :, off] = scale
        else:
            pool[name][pid, :, off] = rows
    pool["phi"][pid, :, off] = phi.permute(0, 2, 1)
    pool["psi"][pid, :, off] = psi.permute(0, 2, 1)


def _own_cache(case, n_pages):
    from first_passage_attention_b200 import FPACache
    return FPACache(n_pages, case["H"], case["D"], page_size=case["page"], dtype=DTYPES[case["type"]],
                    storage=torch.int8 if case["int8"] else None, device=DEVICE)


def prepare(case, seed):
    if case["kind"] == "verify":
        return _prepare_verify(case, seed)
    d = _sequences(case, seed)
    lens, counts = _lens(case), _counts(case)
    st = dict(case=case, table=d["table"], lengths=_int32(lens))
    if own:
        st["cache"] = _own_cache(case, d["n_pages"])
    else:
        st["pool"] = _plain_pool(case, d["n_pages"])
    if case["kind"] == "append":
        # The newest tokens as a model hands them over: views of one fused projection [B, n, 3, H, D].
        n = case["n"]
        qkv = torch.empty(case["B"], n, 3, case["H"], case["D"], dtype=d["k"].dtype, device=DEVICE)
        views = qkv.permute(2, 0, 3, 1, 4)
        views[0].zero_()
        views[1].copy_(d["k"][:, :, :n])
        views[2].copy_(d["v"][:, :, :n])
        st.update(k=views[1], v=views[2], phi=d["phi"][..., :n].contiguous(), psi=d["psi"][..., :n].contiguous(),
                  start=_int32([x - c for x, c in zip(lens, counts)]), counts=_int32(counts))
        return st
    fills = [(d["table"], lens, d["k"], d["v"], d["phi"], d["psi"])]
    if case.get("P"):
        fills.append((d["ptable"][None], [case["P"]], d["pk"], d["pv"], d["pphi"], d["ppsi"]))
    for table, count, k, v, phi, psi in fills:
        start = _int32([0] * len(count))
        if own:
            st["cache"].append(k, v, phi, psi, table, start, _int32(count))
        else:
            _plain_write(st["pool"], table, start, _int32(count), k, v, phi, psi)
    if case["kind"] == "read":
        st["start"] = _int32([x - c for x, c in zip(lens, counts)])
    else:
        st.update(q=d["q"], beta=d["beta"], ptable=d["ptable"], plen=_int32([case["P"]]))
    return st


def _prepare_verify(case, seed):
    """Target and draft probabilities that agree as a draft model's do (about three of four tokens accepted), tokens
    drawn from the draft's, and the random numbers."""
    g = _gen(seed)
    B, n, V = case["B"], case["n"], case["V"]
    logits = 3.0 * torch.randn(B, n + 1, V, generator=g, device=DEVICE)
    q = logits[:, :n].softmax(-1)
    p = logits.add_(0.5 * torch.randn(B, n + 1, V, generator=g, device=DEVICE)).softmax(-1)
    e = torch.empty(B, n, V, device=DEVICE).exponential_(generator=g)
    draft = (q / e).argmax(-1)
    dt = DTYPES[case["type"]]
    return dict(case=case, p=p.to(dt), q=q.to(dt), draft=draft,
                u=torch.rand(B, n, generator=g, device=DEVICE),
                noise=torch.empty(B, V, device=DEVICE).exponential_(generator=g))


# --------------------------------------------------------------------------------------------- the plain forms ----

def _plain_rows(pool, table, start, n, lengths, dtype):
    """Entries at positions start_b .. start_b + n - 1 of each sequence, zero from lengths_b on."""
    page = pool["k"].shape[2]
    pos = start[:, None].long() + torch.arange(n, device=DEVICE)
    ok = pos < lengths[:, None]
    col = (pos // page).clamp(max=table.shape[1] - 1)
    pid = table.long().gather(1, col).clamp(min=0)
    off = pos % page
    out = []
    for name in ("k", "v"):
        x = pool[name][pid, :, off].float()  # [B, n, H, D]
        if name + "s" in pool:
            x = x * pool[name + "s"][pid, :, off][..., None]
        out.append(torch.where(ok[:, :, None, None], x, 0.0).permute(0, 2, 1, 3).to(dtype))
    for name in ("phi", "psi"):
        out.append(torch.where(ok[:, :, None], pool[name][pid, :, off], 0.0).permute(0, 2, 1))
    return out


def _plain_decode(st):
    case, pool, table, lengths = st["case"], st["pool"], st["table"], st["lengths"]
    q, beta = st["q"].float(), st["beta"]
    B, H, n, D = q.shape
    P = case["P"]
    T = table.shape[1] * pool["k"].shape[2]
    inf = float("inf")
    k, v, phi, psi = _plain_rows(pool, table, torch.zeros_like(lengths), T, lengths, torch.float32)
    s = torch.arange(T, device=DEVICE)
    t = lengths[:, None].long() - n + torch.arange(n, device=DEVICE)  # [B, n]
    seen = (s <= t[..., None])[:, None]  # [B, 1, n, T]
    low = torch.where(seen, phi[:, :, None], inf).flip(-1).cummin(-1).values.flip(-1)  # min over u in [s, t]
    after = torch.cat([low[..., 1:], torch.full_like(low[..., :1], inf)], -1)
    bias = beta[:, None, None] * (after - psi[:, :, None]).clamp(max=0.0)
    z = torch.where(seen, q @ k.transpose(-1, -2) * D ** -0.5 + bias, -inf)
    if P:
        pk, pv, pphi, ppsi = _plain_rows(pool, st["ptable"][None], torch.zeros_like(st["plen"]), P, st["plen"],
                                         torch.float32)
        suf = pphi.flip(-1).cummin(-1).values.flip(-1)
        suf = torch.cat([suf[..., 1:], torch.full_like(suf[..., :1], inf)], -1)
        m = torch.minimum(suf[:, :, None], low[..., :1])
        pbias = beta[:, None, None] * (m - ppsi[:, :, None]).clamp(max=0.0)
        rows = q.permute(1, 0, 2, 3).reshape(H, B * n, D)
        pz = (rows @ pk[0].transpose(-1, -2)).view(H, B, n, P).transpose(0, 1) * D ** -0.5 + pbias
        z = torch.cat([pz, z], -1)
    z = z - z.amax(-1, keepdim=True)
    w = torch.exp(z)
    w = w / w.sum(-1, keepdim=True)
    o = w[..., P:] @ v
    if P:
        o = o + (w[..., :P].transpose(0, 1).reshape(H, B * n, P) @ pv[0]).view(H, B, n, D).transpose(0, 1)
    return torch.where((t >= 0)[:, None, :, None], o, 0.0).to(st["q"].dtype)


def _plain_verify(st):
    p, q, draft, u, noise = st["p"].float(), st["q"].float(), st["draft"], st["u"], st["noise"]
    B, n, V = q.shape
    at = draft[..., None]
    ok = u * q.gather(-1, at)[..., 0] < p[:, :n].gather(-1, at)[..., 0]
    accepted = ok.int().cumprod(-1).sum(-1)
    b = torch.arange(B, device=DEVICE)
    pa = p[b, accepted]
    qa = torch.where((accepted < n)[:, None], q[b, accepted.clamp(max=n - 1)], 0.0)
    res = pa - qa
    res = torch.where((res > 0).any(-1, keepdim=True), res, pa)
    score = torch.where(res > 0, res / noise, -1.0)
    best = score.amax(-1, keepdim=True)
    nxt = torch.where(score == best, torch.arange(V, device=DEVICE), V).amin(-1)  # ties go to the lowest index
    i = torch.arange(n + 1, device=DEVICE)
    drafted = torch.cat([draft, draft[:, :1]], -1)
    tokens = torch.where(i < accepted[:, None], drafted, torch.where(i == accepted[:, None], nxt[:, None], -1))
    return accepted.int(), tokens


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from first_passage_attention_b200 import first_passage_decode, verify_draft
        if kind == "verify":
            return verify_draft(state["p"], state["q"], state["draft"], state["u"], state["noise"])
        cache = state["cache"]
        if kind == "decode":
            prefix = dict(prefix_table=state["ptable"], prefix_len=case["P"]) if case["P"] else {}
            return first_passage_decode(state["q"], cache, state["table"], state["lengths"], state["beta"], **prefix)
        if kind == "append":
            cache.append(state["k"], state["v"], state["phi"], state["psi"], state["table"], state["start"],
                         state["counts"])
        return cache.read(state["table"], state["start"], case["n"], state["lengths"])
    if kind == "verify":
        return _plain_verify(state)
    if kind == "decode":
        return _plain_decode(state)
    if kind == "append":
        _plain_write(state["pool"], state["table"], state["start"], state["counts"], state["k"], state["v"],
                     state["phi"], state["psi"])
    return tuple(_plain_rows(state["pool"], state["table"], state["start"], case["n"], state["lengths"],
                             DTYPES[case["type"]]))


# -------------------------------------------------------------------------------------------------------- work ----

def work(case):
    es = {"fp16": 2, "fp32": 4}[case["type"]]
    B, n = case["B"], case["n"]
    if case["kind"] == "verify":
        # A row each of p, q and the noise, and the drafted entries; a subtraction, a division and a comparison.
        return {"bytes": B * (case["V"] * (2 * es + 4) + n * (2 * es + 16) + 4 + 8 * (n + 1)), "flops": 3 * B * case["V"]}
    H, D = case["H"], case["D"]
    stored = 2 * D * (1 if case["int8"] else es) + (8 if case["int8"] else 0) + 8  # a token of a head in the cache
    dense = 2 * D * es + 8
    if case["kind"] in ("append", "read"):
        tokens = sum(_counts(case)) * H
        if case["kind"] == "append":  # in, stored, and read back
            return {"bytes": tokens * (2 * dense + 2 * stored), "flops": tokens * 4 * D}
        return {"bytes": tokens * stored + B * n * H * dense, "flops": tokens * 2 * D}
    keys, rows = sum(_lens(case)) * H, sum(min(n, x) for x in _lens(case)) * H
    P = case["P"]
    return {"bytes": (keys + P * H) * stored + 2 * B * n * H * D * es,
            "flops": 4 * D * (sum(x * min(n, x) for x in _lens(case)) * H + P * rows)}


# ------------------------------------------------------------------------------------------------------- exact ----

def exact(case, seed):
    """The operators' definitions in float64, one sequence (and one query) after the other."""
    if case["kind"] == "verify":
        return _exact_verify(_prepare_verify(case, seed))
    d = _sequences(case, seed)
    lens, counts, n = _lens(case), _counts(case), case["n"]
    if case["kind"] in ("append", "read"):
        B, H, D = case["B"], case["H"], case["D"]
        out = [torch.zeros(B, H, n, D, dtype=torch.float64, device=DEVICE) for _ in range(2)]
        out += [torch.zeros(B, H, n, dtype=torch.float64, device=DEVICE) for _ in range(2)]
        for b in range(B):
            c = counts[b]
            at = slice(0, c) if case["kind"] == "append" else slice(lens[b] - c, lens[b])
            for i, name in enumerate(("k", "v")):
                out[i][b, :, :c] = _exact_stored(case, d[name][b, :, at])
            out[2][b, :, :c] = d["phi"][b, :, at].double()
            out[3][b, :, :c] = d["psi"][b, :, at].double()
        return tuple(out)
    q, beta = d["q"].double(), d["beta"].double()
    o = torch.zeros_like(q)
    pre = {}
    if case["P"]:
        pre = {x: _exact_entry(case, x, d["p" + x][0]) for x in ("k", "v", "phi", "psi")}
    for b, L in enumerate(lens):
        seq = {x: _exact_entry(case, x, d[x][b, :, :L]) for x in ("k", "v", "phi", "psi")}
        if pre:
            seq = {x: torch.cat([pre[x], seq[x]], 1) for x in seq}
        for r in range(n):
            t = L - n + r
            if t < 0:
                continue
            T = case["P"] + t + 1  # keys that this query sees; the last is its own
            least = seq["phi"][:, 1:T].flip(-1).cummin(-1).values.flip(-1) if T > 1 else seq["phi"][:, :0]
            bias = torch.zeros_like(seq["phi"][:, :T])
            bias[:, :T - 1] = torch.minimum(least - seq["psi"][:, :T - 1], torch.zeros_like(least))
            z = torch.einsum("hd,htd->ht", q[b, :, r], seq["k"][:, :T]) / math.sqrt(case["D"]) + beta[:, None] * bias
            o[b, :, r] = torch.einsum("ht,htd->hd", z.softmax(-1), seq["v"][:, :T])
    return o


def _exact_stored(case, x):
    """What the cache stands for: the rows themselves, or their int8 codes times their scale."""
    x = x.double()
    if not case["int8"]:
        return x
    top = x.abs().amax(-1, keepdim=True).clamp(min=1e-300)
    return torch.round(x * 127.0 / top) * (top / 127.0)


def _exact_entry(case, name, x):
    if name in ("phi", "psi"):
        return x.double()
    if case["int8"]:  # attention's input is what the cache holds: codes, and scales in float32
        codes, scale = _quantise(x)
        return codes.double() * scale.double()[..., None]
    return x.double()


def _exact_verify(st):
    p, q, draft = st["p"], st["q"], st["draft"].cpu().tolist()
    u = st["u"].cpu().double().tolist()
    B, n, V = q.shape
    accepted, tokens = [], []
    for b in range(B):
        at = torch.tensor(draft[b], device=DEVICE)
        pd = p[b, :n].double().gather(-1, at[:, None])[:, 0].tolist()
        qd = q[b].double().gather(-1, at[:, None])[:, 0].tolist()
        a = 0
        while a < n and u[b][a] * qd[a] < pd[a]:
            a += 1
        res = p[b, a].double() - (q[b, a].double() if a < n else 0.0)
        if not bool((res > 0).any()):
            res = p[b, a].double()
        score = torch.where(res > 0, res / st["noise"][b].double(), -1.0)
        nxt = int(torch.nonzero(score == score.max())[0, 0])
        accepted.append(a)
        tokens.append(draft[b][:a] + [nxt] + [-1] * (n - a))
    return _int32(accepted), torch.tensor(tokens, device=DEVICE)
