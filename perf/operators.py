"""Cases for timing the serving operators around the packed Linears: the paged
4-bit key/value cache (append with rotary positions, attention, reading rows
back) and the processing of logits before a token is chosen.

`run` computes a case either in plain torch operations (`own` false) or by the
calls that a user makes of drinkme_b200 (`own` true); `exact` computes it from
the definitions in float64.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e6
TOO_SLOW = 6e11  # multiply-adds of `exact` in float64 that stay well under 20 seconds


# --------------------------------------------------------------------------
# the cases

def listed():
    heads8b = dict(nh=32, nkv=8, hd=128, page=64)
    heads32b = dict(nh=64, nkv=8, hd=128, page=64)
    rot = dict(rot=128, interleaved=False, norm=True, dtype="bf16")
    return [
        # one user's decode step: the new token's q, k, v of one layer
        dict(heads8b, **rot, name="append 1 token", op="append", batch=1, q=1, kv=1000),
        # a full decode batch
        dict(heads8b, **rot, name="append 64 sequences", op="append", batch=64, q=1, kv=2000),
        # the chunk of prompts that one prefill forward takes at most
        dict(heads32b, **rot, name="append 4096 prompt tokens", op="append", batch=3, q=1365, kv=1400),
        # a model without q/k norms that rotates half of each head, pairs side by side, fp32 projections
        dict(nh=16, nkv=16, hd=64, page=16, rot=32, interleaved=True, norm=False, dtype="f32",
             name="append 777 tokens, partial", op="append", batch=7, q=111, kv=500),
        # one user's decode step against a short conversation
        dict(heads8b, name="attention 1 x 1000", op="attention", batch=1, q=1, kv=1000, window=0),
        # a decode batch of mixed conversations
        dict(heads8b, name="attention 32 x 8192", op="attention", batch=32, q=1, kv=8192, window=0),
        # one user's decode step against a book
        dict(heads32b, name="attention 1 x 131071", op="attention", batch=1, q=1, kv=131071, window=0),
        # verify batches: four drafted tokens and the one before them
        dict(heads8b, name="attention 8 x 5 tokens", op="attention", batch=8, q=5, kv=4000, window=0),
        # a prompt chunk on top of what the cache holds already
        dict(heads8b, name="attention 2048 prompt tokens", op="attention", batch=1, q=2048, kv=8192, window=0),
        # one user's logits: penalties over the conversation, a few biases, a grammar
        dict(name="logits 1 row", op="logits", batch=1, vocab=151936, history=1000, bias=16, mask=True, dtype="bf16"),
        # a decode batch without a grammar
        dict(name="logits 64 rows", op="logits", batch=64, vocab=151936, history=4000, bias=300, mask=False,
             dtype="f32"),
        # the widest batch, every option
        dict(name="logits 256 rows", op="logits", batch=256, vocab=151936, history=2000, bias=32, mask=True,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "logits"))
    if op == "logits":
        batch = _log(rng, 1, 256)
        return dict(op=op, batch=batch, vocab=_log(rng, 1000, 151936), history=_log(rng, 1, 8000),
                    bias=rng.choice((0, 1, 17, 300)), mask=rng.random() < 0.5, dtype=rng.choice(("bf16", "f32")))
    nh, nkv = rng.choice(((8, 2), (32, 8), (64, 8), (16, 16), (12, 4), (10, 1), (40, 8)))
    hd = rng.choice((64, 128, 128))
    c = dict(op=op, nh=nh, nkv=nkv, hd=hd, page=rng.choice((16, 32, 64, 128, 256)))
    if op == "append":
        batch = _log(rng, 1, 64)
        q = _log(rng, 1, max(1, 4096 // batch)) if rng.random() < 0.6 else 1
        return dict(c, batch=batch, q=q, kv=q + _log(rng, 1, 4000), rot=rng.choice((hd, hd, hd // 2, hd // 4)),
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "f32")))
    kind = rng.choice(("decode", "decode", "verify", "prompt"))
    window = rng.choice((0, 0, 0, _log(rng, 16, 4096)))
    if kind == "prompt":
        q = _log(rng, 9, 2048)
        batch = _log(rng, 1, max(1, 2048 // q))
        return dict(c, nh=min(nh, 32), batch=batch, q=q, kv=q + _log(rng, 1, max(2, 8192 - q)), window=window)
    q = 1 if kind == "decode" else rng.randint(2, 8)
    batch = _log(rng, 1, 32 if kind == "decode" else 8)
    return dict(c, batch=batch, q=q, kv=q + _log(rng, 1, 100000 // (batch * q)), window=window)


def _lengths(case):
    """(new tokens, rows in the cache after them) of each sequence: the first
    has the case's own, the others are spread below them."""
    q, kv = [], []
    for b in range(case["batch"]):
        f = 1.0 - 0.75 * ((b * 0.6180339887) % 1.0)
        new = max(1, int(case["q"] * (1.0 - 0.2 * ((b * 0.381966) % 1.0)))) if case["q"] > 8 else case["q"]
        q.append(new)
        kv.append(max(new, int(case["kv"] * f)))
    return q, kv


def work(case):
    if case["op"] == "logits":
        n = case["batch"] * case["vocab"]
        size = 2 if case["dtype"] == "bf16" else 4
        rows = case["batch"] * (4 * case["history"] + 8 * case["bias"] + 12)
        return {"bytes": 2 * size * n + (n // 8 if case["mask"] else 0) + rows, "flops": 8 * n}
    q, kv = _lengths(case)
    nh, nkv, hd, T = case["nh"], case["nkv"], case["hd"], sum(q)
    held = hd + 8  # codes and scales of a key and a value row
    if case["op"] == "append":
        size = 2 if case["dtype"] == "bf16" else 4
        moved = T * (nh + 2 * nkv) * hd * size + T * nh * hd * 2 + T * nkv * held  # q, k, v in; q and the rows out
        moved += T * nkv * held + T * nkv * 2 * hd * 2 + T * case["rot"] * 4  # the rows read back; the tables
        return {"bytes": moved, "flops": 12 * T * (nh + 2 * nkv) * hd}
    pairs, rows = 0, 0
    for a, n in zip(q, kv):
        w = case["window"] or n
        first = max(0, n - a + 1 - w)
        rows += n - first
        pairs += sum(min(w, n - a + 1 + i) for i in range(a))
    return {"bytes": rows * nkv * held + T * nh * hd * 4, "flops": 4 * pairs * nh * hd}


# --------------------------------------------------------------------------
# inputs

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _paged(case, g, kv):
    """An empty cache's tensors and a page table over shuffled pages; entries
    that no row needs are -1."""
    page, nkv, hd = case["page"], case["nkv"], case["hd"]
    need = [-(-n // page) for n in kv]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV)[: sum(need)].to(torch.int32)
    starts = torch.tensor([0] + need[:-1], device=DEV).cumsum(0)
    col = torch.arange(max(need), device=DEV)[None, :]
    at = starts[:, None] + col
    live = col < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(live, order[at.clamp(max=sum(need) - 1)], torch.full_like(at, -1, dtype=torch.int32))
    codes = torch.empty(pages, nkv, 2, page, hd // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(pages, nkv, page, 4, dtype=torch.bfloat16, device=DEV)
    return codes, scales, table


def _fill(codes, scales, g):
    """What appended rows leave: normal values of one spread per row, keys with
    channels that stand out. Page by page, so that long caches stay cheap."""
    pages, nkv, _, page, half = codes.shape
    step = max(1, (1 << 26) // (nkv * 2 * page * half * 2))
    loud = 1.0 + 3.0 * (torch.rand(nkv, 1, 1, half * 2, generator=g, device=DEV) < 0.05).float()
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, nkv, 2, page, half * 2, generator=g, device=DEV)
        x[:, :, :1] *= loud
        lo, hi = x.amin(-1), x.amax(-1)
        s = ((hi - lo) / 15).to(torch.bfloat16).float()
        m = lo.to(torch.bfloat16).float()
        c = ((x - m[..., None]) / s[..., None]).round().clamp(0, 15).to(torch.uint8)
        codes[p:p + n] = c[..., 0::2] | (c[..., 1::2] << 4)
        scales[p:p + n] = torch.stack((s[:, :, 0], m[:, :, 0], s[:, :, 1], m[:, :, 1]), -1).to(torch.bfloat16)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=dict(case))
    if case["op"] == "logits":
        B, V, N, K = case["batch"], case["vocab"], case["history"], case["bias"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        s["logits"] = (3.0 * torch.randn(B, V, generator=g, device=DEV)).to(dt)
        # a conversation repeats itself: ids by a skewed law, each row of its own length
        u = torch.rand(B, N, generator=g, device=DEV)
        s["history"] = (V * u ** 3).long().clamp(max=V - 1).to(torch.int32)
        s["total"] = (N - (torch.arange(B, device=DEV) * 37) % (N // 2 + 1)).to(torch.int32)
        s["prompt"] = (s["total"].float() * 0.6).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * torch.rand(B, generator=g, device=DEV)
        s["presence"] = 0.5 * torch.rand(B, generator=g, device=DEV)
        s["frequency"] = 0.2 * torch.rand(B, generator=g, device=DEV)
        if K:  # distinct ids, the last few places of a row empty
            off = torch.randint(V, (B, 1), generator=g, device=DEV)
            ids = (off + torch.arange(K, device=DEV)[None, :] * max(1, V // K)) % V
            ids[:, K - K // 8:] = -1
            s["bias_ids"] = ids.to(torch.int32)
            s["bias_values"] = 5.0 * torch.randn(B, K, generator=g, device=DEV)
        if case["mask"]:  # a grammar leaves few tokens; the second row's leaves none
            words = -(-V // 32)
            m = torch.randint(-(1 << 31), 1 << 31, (4, B, words), generator=g, device=DEV).to(torch.int32)
            s["allowed"] = m[0] & m[1] & m[2] & m[3]
            if B > 1:
                s["allowed"][1] = 0
        s["out"] = torch.empty_like(s["logits"])
        return s
    q, kv = _lengths(case)
    nh, nkv, hd, T = case["nh"], case["nkv"], case["hd"], sum(q)
    s["codes"], s["scales"], s["table"] = _paged(case, g, kv)
    s["q_start"] = torch.tensor([0] + q, device=DEV).cumsum(0).to(torch.int32)
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device=DEV)
    s["tokens"], s["max_q"], s["max_kv"] = T, max(q), max(kv)
    if case["op"] == "append":
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # the fused projection's rows: q heads, then k, then v
        s["qkv"] = (0.8 * torch.randn(T, (nh + 2 * nkv) * hd, generator=g, device=DEV)).to(dt)
        inv = 1.0 / THETA ** (torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float32) / case["rot"])
        ang = torch.arange(max(kv), device=DEV, dtype=torch.float32)[:, None] * inv
        s["cos"], s["sin"] = ang.cos(), ang.sin()
        s["qn"] = s["kn"] = None
        if case["norm"]:
            s["qn"] = (1.0 + 0.1 * torch.randn(hd, generator=g, device=DEV)).to(torch.bfloat16)
            s["kn"] = (1.0 + 0.1 * torch.randn(hd, generator=g, device=DEV)).to(torch.bfloat16)
        s["q_out"] = torch.empty(T, nh, hd, dtype=torch.bfloat16, device=DEV)
        s["k_out"] = torch.empty(T, nkv, hd, dtype=torch.bfloat16, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    else:
        _fill(s["codes"], s["scales"], g)
        s["q"] = (1.5 * torch.randn(T, nh, hd, generator=g, device=DEV)).to(torch.bfloat16)
        s["out"] = torch.empty(T, nh, hd, dtype=torch.bfloat16, device=DEV)
    if own:  # the handles that a serving loop keeps: no data is touched
        from drinkme_b200 import kv4

        s["cache"] = kv4.Cache(s["codes"], s["scales"])
        s["batch"] = kv4.Batch(s["table"], s["q_start"], s["kv_len"], tokens=T, max_q=s["max_q"])
    return s


# --------------------------------------------------------------------------
# one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    if op == "append":
        return _plain_append(s)
    if op == "attention":
        return _plain_attention(s)
    return _plain_logits(s)


def _own(s, op):
    from drinkme_b200 import kv4, logits

    c = s["case"]
    if op == "append":
        q, k, v = kv4.split_qkv(s["qkv"], c["nh"], c["nkv"], c["hd"])
        kv4.append(s["cache"], s["batch"], q, k, v, s["cos"], s["sin"], q_norm=s["qn"], k_norm=s["kn"], eps=EPS,
                   interleaved=c["interleaved"], q_out=s["q_out"])
        kv4.read(s["cache"], s["batch"], k_out=s["k_out"], v_out=s["v_out"])
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if op == "attention":
        return kv4.attention(s["cache"], s["batch"], s["q"], window=c["window"], out=s["out"])
    return logits.process(s["logits"], history=s["history"], prompt_len=s["prompt"], total_len=s["total"],
                          repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                          bias_ids=s.get("bias_ids"), bias_values=s.get("bias_values"), allowed=s.get("allowed"),
                          out=s["out"])


def _places(s):
    """(sequence, position) of each new token."""
    t = torch.arange(s["tokens"], device=DEV)
    b = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    return b, s["kv_len"][b] - (s["q_start"][b + 1] - t)


def _pairwise_sum(x):
    """The sum over the last dimension in halving order: this order is part of
    the operator's definition, since 4-bit codes hang on the last bit."""
    n = x.shape[-1]
    return x[..., 0] if n == 1 else _pairwise_sum(x[..., : n // 2] + x[..., n // 2:])


def _rotated(x, w, cos, sin, interleaved):
    """RMSNorm over each head where `w` is given, then the rotation of the
    first 2 * cos.shape[-1] elements. x [T, heads, hd] in float32."""
    if w is not None:
        ss = _pairwise_sum(x * x) * (1.0 / x.shape[-1]) + EPS
        x = x * torch.reciprocal(torch.sqrt(ss))[..., None] * w.float()
    n = cos.shape[-1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    c, d = cos[:, None, :], sin[:, None, :]
    y1, y2 = a * c - b * d, b * c + a * d
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)


def _codes_of(y):
    """(scale, least value, codes) of each row of y, 4 bits a value."""
    lo, hi = y.amin(-1), y.amax(-1)
    m = lo.to(torch.bfloat16).float()
    s = ((hi - lo) * (1.0 / 15.0)).to(torch.bfloat16).float()
    inv = torch.where(s > 0, torch.reciprocal(s), torch.zeros_like(s))
    c = torch.round((y - m[..., None]) * inv[..., None]).clamp(0, 15).to(torch.uint8)
    return s, m, c


def _values_of(codes, scales):
    """float32 values of packed rows: codes [..., hd / 2], scales [..., 2]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return c * scales[..., :1].float() + scales[..., 1:].float()


def _plain_append(s):
    c = s["case"]
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    b, p = _places(s)
    x = s["qkv"].float().view(s["tokens"], nh + 2 * nkv, hd)
    cos, sin = s["cos"][p], s["sin"][p]
    q = _rotated(x[:, :nh], s["qn"], cos, sin, c["interleaved"])
    k = _rotated(x[:, nh:nh + nkv], s["kn"], cos, sin, c["interleaved"])
    sc, m, code = _codes_of(torch.stack((k, x[:, nh + nkv:]), 2))  # [T, nkv, 2, ...]
    at, row = s["table"][b, p // page].long(), p % page
    s["codes"][at, :, :, row] = code[..., 0::2] | (code[..., 1::2] << 4)
    s["scales"][at, :, row] = torch.stack((sc, m), -1).flatten(-2).to(torch.bfloat16)
    held = s["codes"][at, :, :, row]
    two = s["scales"][at, :, row].view(s["tokens"], nkv, 2, 2)
    kv = _values_of(held, two).to(torch.bfloat16)
    return {"q": q.to(torch.bfloat16), "k": kv[:, :, 0].contiguous(), "v": kv[:, :, 1].contiguous()}


def _plain_attention(s):
    c = s["case"]
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    B, Q, L = c["batch"], s["max_q"], -(-s["max_kv"] // page) * page
    at = s["table"][:, : L // page].clamp(min=0).long()
    codes = s["codes"][at].permute(0, 2, 3, 1, 4, 5).reshape(B, nkv, 2, L, hd // 2)
    two = s["scales"][at].permute(0, 2, 1, 3, 4).reshape(B, nkv, L, 4)
    K, V = _values_of(codes[:, :, 0], two[..., :2]), _values_of(codes[:, :, 1], two[..., 2:])
    i = torch.arange(Q, device=DEV)
    qlen = s["q_start"][1:] - s["q_start"][:-1]
    t = (s["q_start"][:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][t].float().view(B, Q, nkv, nh // nkv, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, -1, hd)
    p = (s["kv_len"] - qlen)[:, None] + i  # [B, Q]
    j = torch.arange(L, device=DEV)
    seen = (j <= p[..., None]) & (j < s["kv_len"][:, None, None])
    if c["window"]:
        seen = seen & (j > p[..., None] - c["window"])
    seen = seen[:, None, :, None, :]
    a = torch.matmul(q, K.transpose(2, 3)).view(B, nkv, Q, nh // nkv, L) * (1.0 / math.sqrt(hd))
    a = torch.where(seen, a, torch.full_like(a, -math.inf))
    top = a.amax(-1, keepdim=True)
    a = torch.exp(a - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = a.sum(-1, keepdim=True)
    a = a / torch.where(total == 0, torch.ones_like(total), total)
    V = torch.where((j < s["kv_len"][:, None])[:, None, :, None], V, torch.zeros_like(V))
    o = torch.matmul(a.view(B, nkv, -1, L), V).view(B, nkv, Q, nh // nkv, hd).permute(0, 2, 1, 3, 4)
    b, pos = _places(s)
    return o[b, pos - (s["kv_len"] - qlen)[b]].reshape(s["tokens"], nh, hd).to(torch.bfloat16)


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    n = torch.arange(s["history"].shape[1], device=DEV)[None, :]
    ids = s["history"].long()
    seen = torch.zeros(B, V, device=DEV).scatter_add_(1, ids, (n < s["total"][:, None]).float()) > 0
    made = (n >= s["prompt"][:, None]) & (n < s["total"][:, None])
    count = torch.zeros(B, V, device=DEV).scatter_add_(1, ids, made.float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0).float()
    if "bias_ids" in s:
        bi = s["bias_ids"].long()
        x = x.scatter_add(1, bi.clamp(min=0), torch.where(bi >= 0, s["bias_values"], torch.zeros_like(s["bias_values"])))
    if "allowed" in s:
        v = torch.arange(V, device=DEV)
        bit = (s["allowed"][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        x = torch.where(bit == 1, x, torch.full_like(x, -math.inf))
    return x.to(s["logits"].dtype)


# --------------------------------------------------------------------------
# the same from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attention":
        w = work(case)["flops"]
        return None if w > 2 * TOO_SLOW else _exact_attention(case, s)
    return _exact_logits(case, s)


def _exact_append(case, s):
    nh, nkv, hd, rot = case["nh"], case["nkv"], case["hd"], case["rot"]
    new, kv = _lengths(case)
    pos = torch.cat([torch.arange(n - a, n) for a, n in zip(new, kv)]).to(DEV)
    x = s["qkv"].double().reshape(-1, nh + 2 * nkv, hd)
    head = x[:, : nh + nkv].clone()
    if case["norm"]:
        head *= (head.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        head[:, :nh] *= s["qn"].double()
        head[:, nh:] *= s["kn"].double()
    i = torch.arange(rot // 2, device=DEV)
    one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
    z = torch.complex(head[..., one], head[..., two])
    z = z * torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]
    head[..., one], head[..., two] = z.real.clone(), z.imag.clone()
    rows = torch.stack((head[:, nh:], x[:, nh + nkv:]))
    low = rows.min(-1, keepdim=True).values
    step = ((rows.max(-1, keepdim=True).values - low) / 15).to(torch.bfloat16).double()
    low = low.to(torch.bfloat16).double()
    held = low + step * torch.where(step > 0, (rows - low) / step, rows * 0).round().clamp(0, 15)
    return {"q": head[:, :nh], "k": held[0], "v": held[1]}


def _exact_attention(case, s):
    nh, nkv, hd, page, grp = case["nh"], case["nkv"], case["hd"], case["page"], case["nh"] // case["nkv"]
    out, t = torch.zeros(s["tokens"], nh, hd, dtype=torch.float64, device=DEV), 0
    for b, (a, n) in enumerate(zip(*_lengths(case))):
        pages = s["table"][b, : -(-n // page)].long()
        pos = torch.arange(n - a, n, device=DEV).repeat_interleave(grp)[:, None]
        j = torch.arange(n, device=DEV)[None, :]
        hidden = j > pos
        if case["window"]:
            hidden |= j <= pos - case["window"]
        for h in range(nkv):
            rows = []
            for part in (0, 1):
                byte = s["codes"][pages, h, part].reshape(-1, hd // 2)[:n].int()
                two = s["scales"][pages, h].reshape(-1, 4)[:n].double()
                c = torch.empty(n, hd, dtype=torch.float64, device=DEV)
                c[:, 0::2], c[:, 1::2] = (byte % 16).double(), (byte // 16).double()
                rows.append(two[:, 2 * part + 1, None] + two[:, 2 * part, None] * c)
            q = s["q"][t:t + a, h * grp:(h + 1) * grp].double().reshape(-1, hd)
            logit = (q @ rows[0].T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            out[t:t + a, h * grp:(h + 1) * grp] = (logit.softmax(-1) @ rows[1]).view(a, grp, hd)
        t += a
    return out


def _exact_logits(case, s):
    x = s["logits"].double()
    V = case["vocab"]
    prompt, total = s["prompt"].tolist(), s["total"].tolist()
    for b in range(case["batch"]):
        ids = s["history"][b, : total[b]].long()
        seen = torch.bincount(ids, minlength=V) > 0
        made = torch.bincount(ids[prompt[b]:], minlength=V)
        r = s["repetition"][b].double()
        x[b] = torch.where(seen & (x[b] > 0), x[b] / r, torch.where(seen, x[b] * r, x[b]))
        x[b] -= s["frequency"][b].double() * made + s["presence"][b].double() * (made > 0)
        if case["bias"]:
            live = s["bias_ids"][b] >= 0
            x[b, s["bias_ids"][b][live].long()] += s["bias_values"][b][live].double()
        if case["mask"]:
            words = s["allowed"][b].long()
            bits = (words[:, None] >> torch.arange(32, device=DEV)) & 1
            x[b, bits.reshape(-1)[:V] == 0] = -math.inf
    return x
