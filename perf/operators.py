"""Measured cases of the packed and paged attention operators, the page
operators beside them, and the token log-probability operator.

`own = False` computes each operator in elementary torch operations in 32
bits; `own = True` calls the framework's entry points in `luminaai_amd.ops`.
Sizes come from the presets in `luminaai_amd/config.py` (12:4 heads of 159,
32:8 heads of 128, 8:4 heads of 64, vocabulary 50304, sequences of 2048 and
4096) and the server's default of 8 rows.
"""

import math

import torch

own = False


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a few short prompts that reach the server together (8:4 heads of 64)
        {"name": "packed_prefill_short", "op": "packed", "train": False,
         "heads": 8, "kv_heads": 4, "dim": 64, "lens": "37,1,130,64,0,251",
         "tail": 0},
        # a packed training batch of the 12:4 x 159 preset: documents of
        # uneven length up to the training length of 2048, a ragged end
        {"name": "packed_train_159", "op": "packed", "train": True,
         "heads": 12, "kv_heads": 4, "dim": 159,
         "lens": "2048,1731,2048,95,1,640,1187,429", "tail": 13},
        # a packed training batch of the 32:8 x 128 preset at length 4096
        {"name": "packed_train_128", "op": "packed", "train": True,
         "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "4096,2501,1083,512", "tail": 0},
        # one chat user in the middle of an answer
        {"name": "decode_one", "op": "decode", "heads": 12, "kv_heads": 4,
         "dim": 159, "lens": "2041", "page": 16},
        # the server's eight rows, from a fresh prompt to a full context
        {"name": "decode_batch", "op": "decode", "heads": 32, "kv_heads": 8,
         "dim": 128, "lens": "1,17,400,901,1777,2048,3500,4096", "page": 64},
        # a loaded server: 64 rows, contexts of 1K to 32K
        {"name": "decode_long", "op": "decode", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64,
         "lens": ",".join(str(1001 + 503 * i) for i in range(64))},
        # keys and values of one new token for each of 64 rows
        {"name": "append_decode", "op": "append", "kv_heads": 8, "dim": 128,
         "page": 64, "lens": "1," * 63 + "1", "past": 1500},
        # keys and values of a packed prefill go to their pages
        {"name": "append_prefill", "op": "append", "kv_heads": 4, "dim": 159,
         "page": 16, "lens": "2048,1731,2048,95,1,640,1187,429", "past": 0},
        # a prompt is forked for four answers: its last page is copied
        {"name": "fork_pages", "op": "copy", "layers": 31, "kv_heads": 4,
         "dim": 159, "page": 16, "pool": 60, "pairs": 3},
        # a fragmented pool is compacted
        {"name": "compact_pages", "op": "copy", "layers": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "pool": 700, "pairs": 301},
        # log probabilities of eight rows' sampled tokens, 20 alternatives
        {"name": "logprobs_decode", "op": "logprobs", "train": False,
         "rows": 8, "vocab": 50304, "top_k": 20, "dtype": "float32",
         "masked": True},
        # a policy-gradient step's log probabilities and entropies
        {"name": "logprobs_train", "op": "logprobs", "train": True,
         "rows": 8192, "vocab": 50304, "top_k": 0, "dtype": "bfloat16",
         "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["packed", "packed", "decode", "decode", "append",
                     "copy", "logprobs", "logprobs"])
    heads, kv, dim = rng.choice([(12, 4, 159), (32, 8, 128), (8, 4, 64),
                                 (8, 2, 96), (8, 8, 80), (4, 4, 192),
                                 (40, 10, 128), (2, 1, 64)])
    page = rng.choice([16, 32, 64, 128])
    if op == "packed":
        lens = [_log(rng, 1, 2100) for _ in range(_log(rng, 1, 12))]
        if rng.random() < 0.3:
            lens.append(0)
        return {"op": op, "train": rng.random() < 0.6, "heads": heads,
                "kv_heads": kv, "dim": dim,
                "lens": ",".join(map(str, lens[:4] if heads > 16 else lens)),
                "tail": rng.choice([0, 0, 5])}
    if op == "decode":
        lens = [_log(rng, 1, 20000) for _ in range(_log(rng, 1, 64))]
        return {"op": op, "heads": heads, "kv_heads": kv, "dim": dim,
                "lens": ",".join(map(str, lens)), "page": page}
    if op == "append":
        decode = rng.random() < 0.5
        lens = [1 if decode else _log(rng, 1, 2048)
                for _ in range(_log(rng, 1, 64 if decode else 8))]
        return {"op": op, "kv_heads": kv, "dim": dim, "page": page,
                "lens": ",".join(map(str, lens)),
                "past": rng.randrange(2000)}
    if op == "copy":
        pairs = _log(rng, 1, 120)
        return {"op": op, "layers": rng.randrange(2, 32), "kv_heads": kv,
                "dim": dim, "page": page, "pool": 2 * pairs + 11,
                "pairs": pairs}
    return {"op": op, "train": rng.random() < 0.5, "rows": _log(rng, 1, 4096),
            "vocab": rng.choice([50304, 1024, _log(rng, 700, 100000)]),
            "top_k": rng.choice([0, 1, 5, 20, 32]),
            "dtype": rng.choice(["bfloat16", "float32"]),
            "masked": rng.random() < 0.5}


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _width(dim):
    """Pages hold heads padded to whole 16-byte pieces."""
    return (dim + 7) // 8 * 8


# ------------------------------------------------------------------ inputs
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _tables(lens, page, g, dev):
    """A table row for each sequence over a shuffled pool, and the pool's
    number of pages."""
    need = [max(1, -(-n // page)) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def _pages(total, kv, page, dim, g, dev, layers=None):
    shape = (total, kv, page, _width(dim))
    if layers is not None:
        shape = (layers,) + shape
    t = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    t.normal_(generator=g)
    t[..., dim:] = 0
    return t


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    op = case["op"]
    st = {"case": case, "op": op}

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        t = torch.empty(shape, dtype=dtype, device=dev)
        return t.normal_(generator=g, std=std)

    if op == "packed":
        lens = _lens(case)
        T, H, HKV, D = (sum(lens) + case["tail"], case["heads"],
                        case["kv_heads"], case["dim"])
        # q, k and v are views of one fused projection, as in the model
        qkv = normal(T, (H + 2 * HKV) * D)
        q, k, v = qkv.split([H * D, HKV * D, HKV * D], dim=1)
        st["q"], st["k"], st["v"] = (q.view(T, H, D), k.view(T, HKV, D),
                                     v.view(T, HKV, D))
        st["max_len"] = max(lens)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        if case["train"]:
            st["go"] = normal(T, H, D)
            for n in ("q", "k", "v"):
                st[n] = st[n].detach().requires_grad_(True)
    elif op == "decode":
        lens = _lens(case)
        st["table"], total = _tables(lens, case["page"], g, dev)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        st["q"] = normal(len(lens), case["heads"], case["dim"], std=1.5)
        st["k"] = _pages(total, case["kv_heads"], case["page"], case["dim"],
                         g, dev)
        st["v"] = _pages(total, case["kv_heads"], case["page"], case["dim"],
                         g, dev)
    elif op == "append":
        lens = _lens(case)
        T, past = sum(lens), case["past"]
        st["table"], total = _tables([n + past for n in lens], case["page"],
                                     g, dev)
        ids, pos = [], []
        for b, n in enumerate(lens):
            ids += [b] * n
            pos += range(past, past + n)
        st["ids"] = torch.tensor(ids, dtype=torch.int32, device=dev)
        st["pos"] = torch.tensor(pos, dtype=torch.int32, device=dev)
        HKV, D = case["kv_heads"], case["dim"]
        kv = normal(T, 2 * HKV * D)
        st["nk"], st["nv"] = (t.view(T, HKV, D)
                              for t in kv.split([HKV * D, HKV * D], dim=1))
        st["k"] = _pages(total, HKV, case["page"], D, g, dev)
        st["v"] = _pages(total, HKV, case["page"], D, g, dev)
    elif op == "copy":
        order = torch.randperm(case["pool"], generator=g, device=dev).tolist()
        st["src"] = order[:case["pairs"]]
        st["dst"] = order[case["pairs"]:2 * case["pairs"]]
        for n in ("k", "v"):
            st[n] = _pages(case["pool"], case["kv_heads"], case["page"],
                           case["dim"], g, dev, layers=case["layers"])
    else:
        N, V = case["rows"], case["vocab"]
        dtype = getattr(torch, case["dtype"])
        x = normal(N, V, dtype=dtype, std=2.5)
        tok = torch.randint(0, V, (N,), generator=g, device=dev)
        # most tokens are ones that the model finds likely
        likely = torch.rand(N, generator=g, device=dev) < 0.7
        at = x.gather(1, tok[:, None])
        x.scatter_(1, tok[:, None], at + 9.0 * likely[:, None].to(dtype))
        if case["masked"]:          # a vocabulary's padding is never answered
            x[:, V - 47:] = float("-inf")
            tok.clamp_(max=V - 48)
        tok[::13] = -100            # prompt tokens do not count
        st["x"], st["tok"] = x, tok
        if case["train"]:
            st["x"].requires_grad_(True)
            st["g_lp"] = normal(N, dtype=torch.float32)
            st["g_ent"] = normal(N, dtype=torch.float32, std=0.01)
    return st


# ------------------------------------------------------------- plain forms
def _packed_plain(st):
    """Sequences are padded to the longest; scores, softmax and products are
    whole tensors. The backward pass is written out from the formulas."""
    q, k, v, cu = (st["q"].detach(), st["k"].detach(), st["v"].detach(),
                   st["cu"].long())
    T, H, D = q.shape
    HKV, B, S = k.shape[1], cu.numel() - 1, st["max_len"]
    G, scale = H // HKV, D ** -0.5
    ar = torch.arange(S, device=q.device)
    idx = (cu[:-1, None] + ar).clamp(max=T - 1)                  # [B, S]
    live = ar < (cu[1:] - cu[:-1])[:, None]
    tok = torch.arange(T, device=q.device)
    seq = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    here = (seq < B)[:, None, None]
    seq = seq.clamp(max=B - 1)
    pos = (tok - cu[seq]).clamp(min=0, max=S - 1)

    def padded(t, groups):                      # [B, HKV, groups, S, D]
        t = t.float()[idx] * live[:, :, None, None]
        return t.view(B, S, HKV, groups, D).permute(0, 2, 3, 1, 4).contiguous()

    def packed(t):                              # [B, HKV, g, S, D] -> [T, ., D]
        t = t.permute(0, 3, 1, 2, 4).reshape(B, S, -1, D)
        return (t[seq, pos] * here).to(q.dtype)

    qp, kp, vp = padded(q, G), padded(k, 1), padded(v, 1)
    keep = (ar[None, :] <= ar[:, None]) & live[:, None, :] & live[:, :, None]
    keep = keep[:, None, None]
    s = torch.matmul(qp, kp.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill(~keep, -1e30)
    p = torch.exp(s - s.amax(-1, keepdim=True)) * keep
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    del s
    o = torch.matmul(p, vp)
    if "go" not in st:
        return packed(o)
    go = padded(st["go"], G)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), go).sum(2, True)
    dp = torch.matmul(go, vp.transpose(-1, -2).contiguous())
    ds = p * (dp - (go * o).sum(-1, keepdim=True)) * scale
    del dp, p
    dq = torch.matmul(ds, kp)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), qp).sum(2, True)
    return packed(o), packed(dq), packed(dk), packed(dv)


def _decode_plain(st):
    q, table, lens = st["q"], st["table"].long(), st["lens"].long()
    B, H, D = q.shape
    HKV, page, W = st["k"].shape[1:]
    L = table.shape[1] * page
    k = st["k"][table].permute(0, 2, 1, 3, 4).reshape(B, HKV, L, W)[..., :D]
    v = st["v"][table].permute(0, 2, 1, 3, 4).reshape(B, HKV, L, W)[..., :D]
    qf = q.float().view(B, HKV, H // HKV, D)
    s = torch.matmul(qf, k.float().transpose(-1, -2).contiguous()) * D ** -0.5
    keep = torch.arange(L, device=q.device) < lens[:, None, None, None]
    s = s.masked_fill(~keep, -1e30)
    p = torch.exp(s - s.amax(-1, keepdim=True)) * keep
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return torch.matmul(p, v.float()).view(B, H, D).to(q.dtype)


def _append_plain(st):
    page, D = st["k"].shape[2], st["nk"].shape[-1]
    pos = st["pos"].long()
    pages = st["table"].long()[st["ids"].long(), pos // page]
    for new, pool in ((st["nk"], st["k"]), (st["nv"], st["v"])):
        row = torch.zeros(new.shape[0], new.shape[1], pool.shape[-1],
                          dtype=new.dtype, device=new.device)
        row[..., :D] = new
        pool[pages, :, pos % page] = row
    return st["k"], st["v"]


def _copy_plain(st):
    dev = st["k"].device
    src = torch.tensor(st["src"], device=dev)
    dst = torch.tensor(st["dst"], device=dev)
    for pool in (st["k"], st["v"]):
        pool[:, dst] = pool[:, src]
    return st["k"], st["v"]


def _logprobs_plain(st):
    case = st["case"]
    x, tok = st["x"].detach().float(), st["tok"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    logp = x - m - torch.log(z)
    p = e / z
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    valid = tok != -100
    at = tok.clamp(min=0)[:, None]
    lp = logp.gather(1, at)[:, 0] * valid
    out = [lp, ent]
    if case["top_k"]:
        ids = torch.sort(x, dim=-1, descending=True,
                         stable=True).indices[:, :case["top_k"]]
        out += [logp.gather(1, ids), ids]
    if case["train"]:
        g_lp = (st["g_lp"] * valid)[:, None]
        g_ent = st["g_ent"][:, None]
        inner = torch.where(p > 0, p * (logp + ent[:, None]),
                            torch.zeros_like(p))
        dx = -g_lp * p - g_ent * inner
        dx.scatter_add_(1, at, g_lp)
        out.append(dx.to(st["x"].dtype))
    return out


# --------------------------------------------------------------------- run
def run(state):
    op = state["op"]
    if own:
        from luminaai_amd import ops
        if op == "packed":
            o = ops.flash_attention_packed(state["q"], state["k"], state["v"],
                                           state["cu"])
            if "go" not in state:
                return o
            return (o, *torch.autograd.grad(
                o, (state["q"], state["k"], state["v"]), state["go"]))
        if op == "decode":
            return ops.paged_attention(state["q"], state["k"], state["v"],
                                       state["table"], state["lens"])
        if op == "append":
            ops.paged_kv_append(state["nk"], state["nv"], state["k"],
                                state["v"], state["table"], state["pos"],
                                state["ids"])
            return state["k"], state["v"]
        if op == "copy":
            ops.copy_pages([state["k"], state["v"]], state["src"],
                           state["dst"])
            return state["k"], state["v"]
        case = state["case"]
        r = ops.token_logprobs(state["x"], state["tok"], case["top_k"])
        out = [r.logprobs, r.entropy]
        if case["top_k"]:
            out += [r.top_logprobs, r.top_ids]
        if case["train"]:
            out += torch.autograd.grad([r.logprobs, r.entropy], [state["x"]],
                                       [state["g_lp"], state["g_ent"]])
        return [t.detach() for t in out]
    return {"packed": _packed_plain, "decode": _decode_plain,
            "append": _append_plain, "copy": _copy_plain,
            "logprobs": _logprobs_plain}[op](state)


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "packed":
        lens = _lens(case)
        T, H, HKV, D = (sum(lens) + case["tail"], case["heads"],
                        case["kv_heads"], case["dim"])
        pairs = sum(n * (n + 1) // 2 for n in lens)
        fwd = 2 * T * D * (2 * H + 2 * HKV)
        if not case["train"]:
            return {"bytes": fwd, "flops": 4 * D * H * pairs}
        return {"bytes": fwd + 2 * T * D * (2 * H + 2 * HKV),
                "flops": 14 * D * H * pairs}
    if op == "decode":
        n, B = sum(_lens(case)), len(_lens(case))
        return {"bytes": 2 * case["dim"] * (2 * n * case["kv_heads"]
                                            + 2 * B * case["heads"]),
                "flops": 4 * case["dim"] * case["heads"] * n}
    if op == "append":
        n = sum(_lens(case)) * case["kv_heads"]
        return {"bytes": 2 * 2 * n * (case["dim"] + _width(case["dim"])),
                "flops": 0}
    if op == "copy":
        return {"bytes": 2 * 2 * 2 * case["pairs"] * case["layers"]
                * case["kv_heads"] * case["page"] * _width(case["dim"]),
                "flops": 0}
    n = case["rows"] * case["vocab"]
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": n * size * (2 if case["train"] else 1),
            "flops": n * (12 if case["train"] else 6)}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """Sequence by sequence and row block by row block, in 64 bits."""
    st = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "packed":
        H, HKV, D = case["heads"], case["kv_heads"], case["dim"]
        G, T = H // HKV, st["q"].shape[0]
        names = ["q"] + (["q", "k", "v"] if case["train"] else [])
        outs = [torch.zeros(st[n].shape, dtype=f64, device=st["q"].device)
                for n in names]
        at = 0
        for n in _lens(case):
            sl = slice(at, at + n)
            at += n
            tri = torch.ones(n, n, dtype=torch.bool,
                             device=st["q"].device).tril()
            for h in range(H if n else 0):
                q = st["q"].detach()[sl, h].to(f64)
                k = st["k"].detach()[sl, h // G].to(f64)
                v = st["v"].detach()[sl, h // G].to(f64)
                s = (q @ k.t()) / math.sqrt(D)
                p = torch.softmax(s.masked_fill(~tri, -math.inf), -1)
                outs[0][sl, h] = p @ v
                if case["train"]:
                    g = st["go"][sl, h].to(f64)
                    dp = g @ v.t()
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                    ds = ds / math.sqrt(D)
                    outs[1][sl, h] = ds @ k
                    outs[2][sl, h // G] += ds.t() @ q
                    outs[3][sl, h // G] += p.t() @ g
        return tuple(outs) if case["train"] else outs[0]
    if op == "decode":
        B, H, D = st["q"].shape
        HKV, page = case["kv_heads"], case["page"]
        out = torch.zeros(B, H, D, dtype=f64, device=st["q"].device)
        for b, n in enumerate(_lens(case)):
            pages = st["table"][b, :-(-n // page)].long()
            k = st["k"][pages].transpose(1, 2).reshape(-1, HKV,
                                                       _width(D))[:n, :, :D]
            v = st["v"][pages].transpose(1, 2).reshape(-1, HKV,
                                                       _width(D))[:n, :, :D]
            for h in range(H):
                hk = h // (H // HKV)
                s = (k[:, hk].to(f64) @ st["q"][b, h].to(f64)) / math.sqrt(D)
                out[b, h] = torch.softmax(s, 0) @ v[:, hk].to(f64)
        return out
    if op in ("append", "copy"):
        k, v = st["k"], st["v"]
        if op == "append":
            D, page = case["dim"], case["page"]
            where = (st["table"].long()[st["ids"].long(),
                                        st["pos"].long() // page] * page
                     + st["pos"].long() % page)
            for pool, new in ((k, st["nk"]), (v, st["nv"])):
                flat = pool.transpose(1, 2).contiguous()
                flat.view(-1, *flat.shape[2:])[where, :, :D] = new
                pool.copy_(flat.transpose(1, 2))
        else:
            for pool in (k, v):
                for a, b in zip(st["src"], st["dst"]):
                    pool[:, b].copy_(pool[:, a])
        return k, v
    parts = []
    N, step = case["rows"], 1024
    for a in range(0, N, step):
        x = st["x"].detach()[a:a + step].to(f64)
        tok = st["tok"][a:a + step]
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        ent = -plogp.sum(-1)
        rows = torch.arange(x.shape[0], device=x.device)
        ok = tok >= 0
        lp = torch.where(ok, logp[rows, tok.clamp(min=0)],
                         torch.zeros_like(ent))
        part = [lp, ent]
        if case["top_k"]:
            ids = torch.argsort(x, dim=-1, descending=True, stable=True)
            ids = ids[:, :case["top_k"]]
            part += [torch.take_along_dim(logp, ids, 1), ids]
        if case["train"]:
            gl = st["g_lp"][a:a + step].to(f64) * ok
            ge = st["g_ent"][a:a + step].to(f64)
            dx = (-(gl[:, None] * p)
                  - ge[:, None] * (plogp + p * ent[:, None]))
            dx[rows, tok.clamp(min=0)] += gl
            part.append(dx)
        parts.append(part)
    return [torch.cat(c) for c in zip(*parts)]
