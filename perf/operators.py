"""Measured cases of the decode-step operators: cross attention to an encoder's
states, attention over a cache held in 4 bits (with the rows appended to it)
and the sampling of the next token.

A case is a dict of plain values.  ``prepare`` makes its inputs on the GPU,
``run`` makes one pass: the plain torch form, or the library's calls where the
module's ``own`` is true.  ``exact`` computes the same results in 64 bits.

A page of the 4-bit cache holds, for each key/value head, ``page_tokens`` key
rows and value rows of head_dim / 2 bytes (channel 2i in the low nibble of
byte i), then a (scale, minimum) pair of float16 for each key row and each
value row; a code c stands for minimum + scale * c, where scale is the row's range times 1 / 15 in 32 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------

def cross(name, dtype, batch, heads, kv_heads, head_dim, q_len, k_len, q_var, k_var, padded):
    """q_var / k_var: every length is the same (False) or lognormal up to the given one (True);
    padded: sequences lie q_len / k_len rows apart and a mask leaves some keys out."""
    c = {"kind": "cross", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "q_len": q_len, "k_len": k_len, "q_var": q_var, "k_var": k_var, "padded": padded}
    return dict(c, name=name) if name else c


def kv4(name, dtype, batch, heads, kv_heads, head_dim, page_tokens, q_len, kv_len, kv_var, causal):
    c = {"kind": "kv4", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "page_tokens": page_tokens, "q_len": q_len, "kv_len": kv_len, "kv_var": kv_var, "causal": causal}
    return dict(c, name=name) if name else c


def append(name, dtype, batch, kv_heads, head_dim, page_tokens, count, first):
    c = {"kind": "append", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim,
         "page_tokens": page_tokens, "count": count, "first": first}
    return dict(c, name=name) if name else c


def sample(name, dtype, rows, vocab, mode):
    """mode: which settings the rows have: "mixed" (every row its own), "top_p", "top_k" or "plain"."""
    c = {"kind": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "mode": mode}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decode step's cross attention of a small server: 64 sentences, the benchmark model's heads.
        cross("cross_token_f32", "f32", 64, 8, 8, 64, 1, 256, False, True, False),
        # Scoring given translations of a batch of sentences: every target token at once, packed.
        cross("cross_score_bf16", "bf16", 256, 8, 8, 64, 256, 256, True, True, False),
        # A padded batch with its attention mask, heads of 48 channels (d = 384 with 8 heads).
        cross("cross_padded_f16", "f16", 64, 8, 8, 48, 200, 255, True, True, True),
        # Whole documents: thousands of target tokens against thousands of source states.
        cross("cross_document_bf16", "bf16", 2, 16, 4, 128, 4096, 8192, False, False, False),
        # One sentence alone, where latency counts.
        kv4("kv4_one_f32", "f32", 1, 8, 8, 64, 16, 1, 230, False, False),
        # A decode step's self attention over 1,024 sentences in flight.
        kv4("kv4_token_f32", "f32", 1024, 8, 8, 64, 16, 1, 256, True, False),
        # A few streams over long caches, with shared key/value heads.
        kv4("kv4_long_bf16", "bf16", 8, 32, 8, 128, 16, 1, 65536, False, False),
        # A chunk of given tokens against the cache that they were just appended to.
        kv4("kv4_chunk_f16", "f16", 16, 16, 2, 64, 32, 33, 4001, True, True),
        # The step's new token of every sentence in flight.
        append("append_token_f32", "f32", 1024, 8, 64, 16, 1, 131),
        # Prompts put into the cache.
        append("append_prompt_bf16", "bf16", 32, 8, 128, 16, 4090, 3),
        # The next token of a handful of streams.
        sample("sample_few_f32", "f32", 8, 32000, "mixed"),
        # The next token of 1,024 sentences in flight, each with its own settings.
        sample("sample_step_f32", "f32", 1024, 32000, "mixed"),
    ]


def spread(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["cross", "cross", "kv4", "kv4", "append", "sample", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "sample":
        vocab = spread(rng, 1000, 152000)
        return sample(None, dtype, spread(rng, 1, max(1, min(1024, 32768000 // vocab))), vocab,
                      rng.choice(["mixed", "mixed", "top_p", "top_k", "plain"]))
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 1, 2, 4, 7, 8])
    heads, head_dim = kv_heads * group, rng.choice([32, 48, 64, 64, 80, 96, 128, 128])
    page_tokens = rng.choice([8, 16, 32])
    if kind == "append":
        batch = spread(rng, 1, 1024)
        count = rng.choice([1, spread(rng, 1, max(1, min(4096, (1 << 25) // (batch * kv_heads * head_dim))))])
        return append(None, dtype, batch, kv_heads, head_dim, page_tokens, count, rng.randrange(0, 300))
    if kind == "kv4":
        batch = spread(rng, 1, 512)
        q_len = rng.choice([1, 1, spread(rng, 1, 64)])
        most = (1 << 28) // (batch * max(kv_heads * head_dim, heads * q_len))
        kv_len = spread(rng, max(16, q_len), max(64, min(65536, most)))
        return kv4(None, dtype, batch, heads, kv_heads, head_dim, page_tokens, q_len, kv_len, rng.random() < 0.6,
                   rng.random() < 0.5)
    k_len = spread(rng, 1, 4096)
    q_len = rng.choice([1, spread(rng, 1, 2048)])
    # f32 products have no fast unit: an f32 case is held to a sixteenth of the 16-bit ones' work
    most = (1 << 36) // (heads * head_dim * q_len * k_len) // (16 if dtype == "f32" else 1)
    batch = spread(rng, 1, max(1, min(256, most, (1 << 28) // (heads * q_len * k_len) or 1)))
    return cross(None, dtype, batch, heads, kv_heads, head_dim, q_len, k_len, rng.random() < 0.6, rng.random() < 0.6,
                 rng.random() < 0.3)


# ---- inputs -----------------------------------------------------------------

def lengths(n, most, vary, least=1, rs=None):
    """Sentence-like lengths: lognormal (median 24 tokens, or an eighth of longer ranges), or all the same.
    A case always has the same ones; rs puts them in another order."""
    if not vary:
        return np.full(n, most, np.int64)
    mid = max(24.0, most / 8) if most > 256 else min(24.0, max(1.0, most / 2))
    drawn = np.random.RandomState(n * 31 + most).normal(math.log(mid), 0.8, n)
    got = np.clip(np.round(np.exp(drawn)), least, most).astype(np.int64)
    return got if rs is None else rs.permutation(got)


def normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))
    return {"cross": prepare_cross, "kv4": prepare_kv4, "append": prepare_append, "sample": prepare_sample}[
        case["kind"]](case, gen, rs)


def prepare_cross(c, gen, rs):
    dtype, b = DTYPES[c["dtype"]], c["batch"]
    q_len = lengths(b, c["q_len"], c["q_var"], rs=rs)
    k_len = lengths(b, c["k_len"], c["k_var"], rs=rs)
    if c["padded"]:
        q_start, k_start = np.arange(b) * c["q_len"], np.arange(b) * c["k_len"]
        q_rows, k_rows = b * c["q_len"], b * c["k_len"]
    else:
        q_start, k_start = np.cumsum(q_len) - q_len, np.cumsum(k_len) - k_len
        q_rows, k_rows = int(q_len.sum()), int(k_len.sum())
    mask = None
    if c["padded"]:
        live = rs.rand(k_rows) < 0.9
        live[k_start[0]:k_start[0] + k_len[0]] = b == 1  # a sentence of which nothing is left
        mask = torch.from_numpy(live.astype(np.uint8)).cuda()
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    return {"case": c, "q": normal(gen, (q_rows, h, d), dtype), "k": normal(gen, (k_rows, hk, d), dtype),
            "v": normal(gen, (k_rows, hk, d), dtype), "out": torch.zeros((q_rows, h, d), dtype=dtype, device="cuda"),
            "lse": torch.zeros((q_rows, h), device="cuda"), "q_start": ints(q_start), "q_len": ints(q_len),
            "k_start": ints(k_start), "k_len": ints(k_len), "mask": mask, "max_q": int(q_len.max()),
            "max_k": int(k_len.max()), "scale": d ** -0.5, "call": None}


def quantized(x):
    """Rows [..., head_dim] in 32 bits -> codes (uint8) and the float16 pair (scale, minimum) of each row."""
    low, high = x.amin(-1), x.amax(-1)
    minimum = low.to(torch.float16)
    scale = ((high - minimum.float()) * (1.0 / 15.0)).to(torch.float16)
    t = (x.double() - minimum.double().unsqueeze(-1)) / scale.double().unsqueeze(-1)
    codes = torch.round(t).clamp(0, 15)
    return torch.where(scale.unsqueeze(-1) > 0, codes, torch.zeros_like(codes)).to(torch.uint8), torch.stack(
        [scale, minimum], -1)


def prepare_kv4(c, gen, rs):
    dtype, b, t = DTYPES[c["dtype"]], c["batch"], c["page_tokens"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    kv_len = lengths(b, c["kv_len"], c["kv_var"], c["q_len"], rs)
    per_seq = -(-int(kv_len.max()) // t)
    used = -(-kv_len // t)
    n_pages = int(used.sum()) + 3
    table = np.full((b, per_seq), -1, np.int64)
    table[np.arange(per_seq)[None, :] < used[:, None]] = rs.permutation(n_pages)[:int(used.sum())]
    # rows as they come from quantizing normal values: codes about their row's middle, steps of a fifteenth of its range
    pages = torch.empty((n_pages, hk, t * (d + 8)), dtype=torch.uint8, device="cuda")
    nibbles = lambda: (torch.randn((n_pages, hk, 2 * t * d // 2), generator=gen, device="cuda") * 3.2 + 8).clamp_(0, 15).to(torch.uint8)  # noqa: E731
    codes = nibbles()
    codes |= nibbles() << 4
    pages[:, :, :t * d] = codes
    params = torch.rand((n_pages, hk, 2 * t, 2), generator=gen, device="cuda") * 0.2
    params += torch.tensor([0.25, -2.5], device="cuda")
    pages[:, :, t * d:] = params.to(torch.float16).view(torch.uint8).view(n_pages, hk, 8 * t)
    q_rows = b * c["q_len"]
    return {"case": c, "pages": pages, "table": ints(table), "kv_len": ints(kv_len),
            "q": normal(gen, (q_rows, h, d), dtype), "out": torch.zeros((q_rows, h, d), dtype=dtype, device="cuda"),
            "lse": torch.zeros((q_rows, h), device="cuda"), "q_start": ints(np.arange(b) * c["q_len"]),
            "q_len": ints(np.full(b, c["q_len"])), "max_kv": int(kv_len.max()), "scale": d ** -0.5, "call": None}


def prepare_append(c, gen, rs):
    dtype, b, t = DTYPES[c["dtype"]], c["batch"], c["page_tokens"]
    hk, d, n = c["kv_heads"], c["head_dim"], c["count"]
    per_seq = -(-(c["first"] + n) // t)
    n_pages = b * per_seq + 1
    rows = b * n
    return {"case": c, "k": normal(gen, (rows, hk, d), dtype), "v": normal(gen, (rows, hk, d), dtype) * 0.7,
            "pages": torch.zeros((n_pages, hk, t * (d + 8)), dtype=torch.uint8, device="cuda"),
            "table": ints(rs.permutation(n_pages)[:b * per_seq].reshape(b, per_seq)),
            "start": ints(np.arange(b) * n), "count": ints(np.full(b, n)), "first": ints(np.full(b, c["first"])),
            "k_back": torch.zeros((rows, hk, d), dtype=dtype, device="cuda"),
            "v_back": torch.zeros((rows, hk, d), dtype=dtype, device="cuda"), "call": None}


def prepare_sample(c, gen, rs):
    dtype, r, v = DTYPES[c["dtype"]], c["rows"], c["vocab"]
    # A model's logits: a bell of unlikely tokens and a few that stand out.
    x = torch.randn((r, v), generator=gen, device="cuda") * 1.6
    x += 14.0 * torch.rand((r, v), generator=gen, device="cuda").pow_(400.0)
    x[:, 1] = -math.inf  # a token that is never to be generated
    mode = c["mode"]
    temperature = rs.uniform(0.5, 1.3, r) if mode in ("mixed", "plain") else np.ones(r)
    temperature[rs.rand(r) < 0.1 * (mode == "mixed")] = 0.0
    top_k = np.where(rs.rand(r) < 0.5, rs.randint(1, 200, r), 0) if mode == "mixed" else np.full(r, 50 * (mode == "top_k"))
    top_p = np.where(rs.rand(r) < 0.7, rs.uniform(0.3, 0.99, r), 1.0) if mode == "mixed" else np.full(
        r, 0.9 if mode == "top_p" else 1.0)
    min_p = np.where(rs.rand(r) < 0.3, rs.uniform(0.01, 0.2, r), 0.0) if mode == "mixed" else np.zeros(r)
    f32 = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    return {"case": c, "logits": x.to(dtype), "temperature": f32(temperature), "top_k": ints(top_k), "top_p": f32(top_p),
            "min_p": f32(min_p), "uniform": f32(rs.randint(0, 1 << 24, r) / float(1 << 24)),
            "tokens": torch.zeros(r, dtype=torch.int32, device="cuda"), "probs": torch.zeros(r, device="cuda"), "call": None}


# ---- one pass ---------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        if s["call"] is None:
            s["call"] = {"cross": own_cross, "kv4": own_kv4, "append": own_append, "sample": own_sample}[kind](s)
        return s["call"]()
    return {"cross": plain_cross, "kv4": plain_kv4, "append": plain_append, "sample": plain_sample}[kind](s)


def padded_rows(x, start, n):
    """Rows start[b] + 0..n of packed x, [batch, n, ...] in 32 bits; the rows behind a sequence are whatever is there."""
    at = (start.long()[:, None] + torch.arange(n, device="cuda")).clamp(max=x.shape[0] - 1)
    return x[at].float(), at


def attend(q, k, v, live, scale):
    """q [b, m, h, d], k and v [b, n, hk, d], live [b, 1 or m, n] -> (out [b, m, h, d], lse [b, m, h])."""
    b, m, h, d = q.shape
    n, hk = k.shape[1:3]
    q = q.view(b, m, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)).view(b, hk, h // hk, m, n) * scale
    x = x.masked_fill(~live[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(b, hk, -1, n), v.permute(0, 2, 1, 3)).view(b, hk, h // hk, m, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    lse = torch.log(total) + top
    return out.permute(0, 3, 1, 2, 4).reshape(b, m, h, d), lse[..., 0].permute(0, 3, 1, 2).reshape(b, m, h)


def plain_cross(s):
    q, q_at = padded_rows(s["q"], s["q_start"], s["max_q"])
    k, k_at = padded_rows(s["k"], s["k_start"], s["max_k"])
    v, _ = padded_rows(s["v"], s["k_start"], s["max_k"])
    live = torch.arange(s["max_k"], device="cuda") < s["k_len"][:, None]
    if s["mask"] is not None:
        live &= s["mask"][k_at] != 0
    v = v.masked_fill(~live[..., None, None], 0.0)
    o, l = attend(q, k, v, live[:, None], s["scale"])
    there = torch.arange(s["max_q"], device="cuda") < s["q_len"][:, None]
    out, lse = torch.zeros_like(s["out"]), torch.zeros_like(s["lse"])
    out[q_at[there]] = o[there].to(out.dtype)
    lse[q_at[there]] = l[there]
    return out, lse


def unpacked(pages, table, t, d):
    """The pages of `table` [b, p] as rows in 32 bits: keys and values [b, p * t, hk, d]."""
    b, p = table.shape
    x = pages[table.long().clamp(min=0)]  # [b, p, hk, t * (d + 8)]
    hk = x.shape[2]
    params = x[..., t * d:].contiguous().view(torch.float16).float().view(b, p, hk, 2, t, 1, 2)
    codes = x[..., :t * d].reshape(b, p, hk, 2, t, d // 2)
    codes = torch.stack([codes & 15, codes >> 4], -1).view(b, p, hk, 2, t, d)
    rows = params[..., 1] + params[..., 0] * codes.float()
    rows = rows.permute(3, 0, 1, 4, 2, 5).reshape(2, b, p * t, hk, d)
    return rows[0], rows[1]


def plain_kv4(s):
    c = s["case"]
    b, m, d = c["batch"], c["q_len"], c["head_dim"]
    k, v = unpacked(s["pages"], s["table"], c["page_tokens"], d)
    at = torch.arange(k.shape[1], device="cuda")
    last = s["kv_len"][:, None] - (m - 1 - torch.arange(m, device="cuda") if c["causal"] else torch.zeros(1, device="cuda", dtype=torch.int64))
    live = at < last[..., None]  # [b, m or 1, n]
    v = v.masked_fill(~live.any(1)[..., None, None], 0.0)
    o, l = attend(s["q"].float().view(b, m, -1, d), k, v, live, s["scale"])
    return o.reshape(s["out"].shape).to(s["out"].dtype), l.reshape(s["lse"].shape)


def plain_append(s):
    c = s["case"]
    t, d, n = c["page_tokens"], c["head_dim"], c["count"]
    at = c["first"] + torch.arange(n, device="cuda")
    page = s["table"].long()[:, at // t].reshape(-1)  # [b * n]
    slot = (at % t).repeat(c["batch"])
    back = []
    both = s["pages"]
    params = both[..., t * d:].view(torch.float16).view(both.shape[0], -1, 2, t, 2)
    codes = both[..., :t * d].view(both.shape[0], -1, 2, t, d // 2)
    ck, pk = quantized(s["k"].float())
    cv, pv = quantized(s["v"].float())
    codes[page, :, 0, slot] = ck[..., 0::2] | ck[..., 1::2] << 4
    codes[page, :, 1, slot] = cv[..., 0::2] | cv[..., 1::2] << 4
    params[page, :, 0, slot] = pk
    params[page, :, 1, slot] = pv
    back = [codes[page, :, i, slot] for i in (0, 1)], [params[page, :, i, slot].float() for i in (0, 1)]
    k, v = (p[..., 1:] + p[..., :1] * torch.stack([x & 15, x >> 4], -1).view(-1, c["kv_heads"], d).float()
            for x, p in zip(*back))
    return k.to(s["k"].dtype), v.to(s["v"].dtype)


def plain_sample(s):
    x, vocab = s["logits"], s["logits"].shape[1]
    column = lambda n: s[n].double()[:, None]  # noqa: E731
    value, order = torch.sort(x.float(), dim=1, descending=True, stable=True)
    value, rank = value.double(), torch.arange(vocab, device="cuda")
    temperature, top = column("temperature"), value[:, :1]
    greedy = temperature == 0
    weight = torch.exp((value - top) / torch.where(greedy, 1.0, temperature))
    keep = value > -math.inf
    limit = s["top_k"].long()[:, None]
    limit = torch.where((limit <= 0) | (limit > vocab), vocab, limit)
    keep &= rank < torch.where(greedy, 1, limit)
    weight = torch.where(keep, weight, 0.0)
    before = torch.cumsum(weight, 1) - weight
    keep &= (rank == 0) | (column("top_p") >= 1) | (before < column("top_p") * weight.sum(1, keepdim=True))
    keep &= (rank == 0) | (weight >= column("min_p"))
    weight = torch.where(keep, weight, 0.0)
    by_id = torch.zeros_like(weight).scatter_(1, order, weight)
    running = torch.cumsum(by_id, 1)
    total = running[:, -1:]
    hit = (running > column("uniform") * total) & (by_id > 0)
    token = hit.to(torch.uint8).argmax(1)
    return token.int(), (by_id.gather(1, token[:, None]) / total)[:, 0].float()


# ---- the library's calls ----------------------------------------------------

def library():
    import os
    import sys
    package = os.path.join(os.getcwd(), "marian-edge_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from marian_cuda import _lib
    return _lib, _lib.load()


def bind(L, function, result, *args):
    """A pass: the call on torch's current stream, which raises where the library refuses it."""
    def call():
        L.check(function(*args, torch.cuda.current_stream().cuda_stream))
        return result
    return call


def strides(**tensors):
    return {"%s_%s_stride" % (n, what): t.stride(i) for n, t in tensors.items() for i, what in enumerate(("row", "head"))}


def kinds(L):
    return {torch.float32: L.MC_F32, torch.float16: L.MC_F16, torch.bfloat16: L.MC_BF16}


def pointers(**tensors):
    return {n: t.data_ptr() for n, t in tensors.items() if t is not None}


def with_workspace(s, args, need):
    s["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_bytes = s["workspace"].data_ptr(), need


def own_cross(s):
    L, lib = library()
    c, ref = s["case"], L.C.byref
    a = L.CrossAttentionArgs(
        **pointers(q=s["q"], k=s["k"], v=s["v"], out=s["out"], lse=s["lse"], q_start=s["q_start"], q_len=s["q_len"],
                   k_start=s["k_start"], k_len=s["k_len"], key_mask=s["mask"]),
        **strides(q=s["q"], k=s["k"], v=s["v"], out=s["out"]), q_rows=s["q"].shape[0], k_rows=s["k"].shape[0],
        dtype=kinds(L)[s["q"].dtype], batch=c["batch"], heads=c["heads"], kv_heads=c["kv_heads"],
        head_dim=c["head_dim"], max_q_len=s["max_q"], max_k_len=s["max_k"], scale=s["scale"])
    with_workspace(s, a, lib.mc_cross_attention_workspace(ref(a)))
    return bind(L, lib.mc_cross_attention, (s["out"], s["lse"]), ref(a))


def own_cache(L, s):
    c = s["case"]
    return L.Kv4Cache(pages=s["pages"].data_ptr(), page_table=s["table"].data_ptr(), n_pages=s["pages"].shape[0],
                      page_tokens=c["page_tokens"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], batch=c["batch"],
                      pages_per_seq=s["table"].shape[1])


def own_kv4(s):
    L, lib = library()
    c, ref = s["case"], L.C.byref
    a = L.Kv4AttentionArgs(
        **pointers(q=s["q"], out=s["out"], lse=s["lse"], q_start=s["q_start"], q_len=s["q_len"], kv_len=s["kv_len"]),
        **strides(q=s["q"], out=s["out"]), q_rows=s["q"].shape[0], dtype=kinds(L)[s["q"].dtype], heads=c["heads"],
        max_q_len=c["q_len"], max_kv_len=s["max_kv"], causal=int(c["causal"]), scale=s["scale"])
    cache = own_cache(L, s)
    with_workspace(s, a, lib.mc_kv4_attention_workspace(ref(cache), ref(a)))
    return bind(L, lib.mc_kv4_attention, (s["out"], s["lse"]), ref(cache), ref(a))


def own_append(s):
    L, lib = library()
    c, ref = s["case"], L.C.byref
    rows = lambda k, v: L.Kv4Rows(  # noqa: E731
        **pointers(k=k, v=v, start=s["start"], count=s["count"], first=s["first"]), **strides(k=k, v=v),
        rows=k.shape[0], dtype=kinds(L)[k.dtype], max_count=c["count"])
    cache, new, back = own_cache(L, s), rows(s["k"], s["v"]), rows(s["k_back"], s["v_back"])
    put = bind(L, lib.mc_kv4_append, None, ref(cache), ref(new))
    get = bind(L, lib.mc_kv4_read, (s["k_back"], s["v_back"]), ref(cache), ref(back))

    def call():
        put()
        return get()
    return call


def own_sample(s):
    L, lib = library()
    x = s["logits"]
    a = L.SampleArgs(
        **pointers(logits=x, temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                   uniform=s["uniform"], tokens=s["tokens"], probs=s["probs"]),
        row_stride=x.stride(0), dtype=kinds(L)[x.dtype], rows=x.shape[0], vocab=x.shape[1])
    return bind(L, lib.mc_sample, (s["tokens"], s["probs"]), L.C.byref(a))


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    c, size = case, {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * size + 28), "flops": 4 * c["rows"] * c["vocab"]}
    hk, d, b = c["kv_heads"], c["head_dim"], c["batch"]
    if c["kind"] == "append":  # the rows in, the cache written and read, the rows back
        values = 2 * b * c["count"] * hk
        return {"bytes": values * (2 * d * size + 2 * (d // 2 + 4)), "flops": 8 * values * d}
    h = c["heads"]
    if c["kind"] == "kv4":
        keys = float(lengths(b, c["kv_len"], c["kv_var"], c["q_len"]).sum())
        rows = b * c["q_len"]
        return {"bytes": keys * hk * (d + 8) + rows * h * (2 * d * size + 4), "flops": 4 * keys * c["q_len"] * h * d}
    q, k = (float(lengths(b, c[n + "_len"], c[n + "_var"]).mean()) for n in ("q", "k"))
    return {"bytes": b * (k * 2 * hk * d * size + q * h * (2 * d * size + 4)), "flops": 4 * b * q * k * h * d}


# ---- the same in 64 bits ----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"cross": exact_cross, "kv4": exact_kv4, "append": exact_append, "sample": exact_sample}[case["kind"]](s)


def softmax_average(q, k, v, seen, scale):
    """One sequence: q [m, h, d], k and v [n, hk, d], seen [m, n] in 64 bits, head by head."""
    m, h, _ = q.shape
    group = h // k.shape[1]
    out, lse = torch.zeros_like(q), torch.full((m, h), -math.inf, dtype=torch.float64, device="cuda")
    for j in range(h):
        x = torch.einsum("md,nd->mn", q[:, j], k[:, j // group]) * scale
        x[~seen] = -math.inf
        lse[:, j] = torch.logsumexp(x, 1)
        some = seen.any(1)
        out[some, j] = torch.softmax(x[some], 1) @ v[:, j // group]
    return out, lse


def exact_cross(s):
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    for q0, m, k0, n in zip(*(s[x].tolist() for x in ("q_start", "q_len", "k_start", "k_len"))):
        seen = torch.ones(n, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][k0:k0 + n] != 0
        k, v = (s[x][k0:k0 + n][seen].double() for x in ("k", "v"))
        if k.shape[0]:
            every = torch.ones((m, k.shape[0]), dtype=torch.bool, device="cuda")
            out[q0:q0 + m], lse[q0:q0 + m] = softmax_average(s["q"][q0:q0 + m].double(), k, v, every, s["scale"])
        else:
            lse[q0:q0 + m] = -math.inf
    return out, lse


def rows_of(block, t, d):
    """One head's pages [p, t * (d + 8)] as keys and values [p * t, d] in 64 bits."""
    halves = block[:, t * d:].contiguous().view(torch.float16).double().view(-1, 2, t, 2)
    both = []
    for i in (0, 1):
        byte = block[:, i * t * d // 2:(i + 1) * t * d // 2].reshape(-1, t, d // 2).long()
        code = torch.empty(byte.shape[0], t, d, dtype=torch.float64, device="cuda")
        code[..., 0::2], code[..., 1::2] = byte % 16, byte // 16
        both.append((halves[:, i, :, 1:] + halves[:, i, :, :1] * code).reshape(-1, d))
    return both


def exact_kv4(s):
    c = s["case"]
    t, d, m = c["page_tokens"], c["head_dim"], c["q_len"]
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["kv_len"].tolist()):
        ids = s["table"][i, :-(-n // t)].long()
        heads = [rows_of(s["pages"][ids, j], t, d) for j in range(c["kv_heads"])]
        k, v = (torch.stack([x[w][:n] for x in heads], 1) for w in (0, 1))
        last = n - m + 1 + torch.arange(m, device="cuda") if c["causal"] else torch.full((m,), n, device="cuda")
        seen = torch.arange(n, device="cuda")[None, :] < last[:, None]
        at = slice(i * m, (i + 1) * m)
        out[at], lse[at] = softmax_average(s["q"][at].double(), k, v, seen, s["scale"])
    return out, lse


def exact_append(s):
    back = []
    for x in (s["k"].double(), s["v"].double()):
        low = x.min(-1, keepdim=True).values.half().double()
        step = ((x.max(-1, keepdim=True).values - low).float() * (1.0 / 15.0)).half().double()
        code = torch.where(step > 0, torch.round((x - low) / step.clamp(min=1e-30)), torch.zeros_like(x))
        back.append(low + step * code.clamp(0, 15))
    return tuple(back)


def exact_sample(s):
    x = s["logits"].float().cpu().numpy().astype(np.float64)
    t, k, p, m, u = (s[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
    tokens, probs = np.zeros(len(x), np.int32), np.zeros(len(x))
    for i, row in enumerate(x):
        ids = np.lexsort((np.arange(row.size), -row))
        ids = ids[row[ids] > -np.inf]
        if t[i] == 0:
            tokens[i], probs[i] = ids[0], 1.0
            continue
        if 0 < k[i] < ids.size:
            ids = ids[:int(k[i])]
        w = np.exp((row[ids] - row[ids[0]]) / t[i])
        if p[i] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), p[i] * w.sum()))
            ids, w = ids[:n], w[:n]
        ids, w = ids[w >= m[i]], w[w >= m[i]]
        by_id = np.argsort(ids)
        sums = np.cumsum(w[by_id])
        at = by_id[min(int(np.searchsorted(sums, u[i] * sums[-1], side="right")), ids.size - 1)]
        tokens[i], probs[i] = ids[at], w[at] / w.sum()
    return torch.from_numpy(tokens), torch.from_numpy(probs)
