"""The decode-step operators together, as a decoder that samples several
translations of each source uses them: every step appends the new token's keys
and values to the 4-bit cache, attends over it, attends to the encoder's states
(which the translations of one source share) and draws the next token.

Every operator's result is compared with the 64-bit form of its definition on
the inputs that it was given, so no error adds up; tolerances as in each
operator's own tests.
"""
import ctypes as C
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from marian_cuda import _lib as L  # noqa: E402
from test_cross_attention import arguments as cross_arguments, attend as cross_attend  # noqa: E402
from test_kv4 import Cache, attend as kv_attend, ints, quantize, rows_struct, score_error, status_bits  # noqa: E402
from test_sample import reference as sample_reference  # noqa: E402

HEADS, DIM, VOCAB, STEPS = 4, 48, 977, 21
D = HEADS * DIM


def f64(x):
    return x.float().cpu().numpy().astype(np.float64)


class Decoder:
    """One attention layer of random weights in f32, over the library's operators."""

    def __init__(self, src_len, copies, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.embed = rnd(VOCAB, D)
        self.w = {n: rnd(D, D) / D ** 0.5 for n in ("q", "k", "v", "o", "cq")}
        self.out = rnd(D, VOCAB) * 3 / D ** 0.5
        self.batch = len(src_len) * copies
        src = int(np.sum(src_len))
        self.enc_k, self.enc_v = rnd(src, HEADS, DIM), rnd(src, HEADS, DIM)
        start = np.cumsum(src_len) - src_len
        self.k_start, self.k_len = np.repeat(start, copies), np.repeat(src_len, copies)
        self.cache = Cache(self.batch, -(-STEPS // 8), 8, HEADS, DIM, fill=0xFF)
        self.uniform = torch.rand(STEPS, self.batch, generator=g, device="cuda")
        self.temperature = torch.linspace(0.0, 1.2, self.batch, device="cuda")
        self.one = ints(np.ones(self.batch))
        self.rows = ints(np.arange(self.batch))
        self.source = [ints(self.k_start), ints(self.k_len)]

    def step(self, t, tokens, stream):
        lib, b = L.load(), self.batch
        x = self.embed[tokens.long()]
        q, k, v = ((x @ self.w[n]).view(b, HEADS, DIM) for n in ("q", "k", "v"))
        cache = self.cache.struct()
        new = rows_struct(k, v, np.arange(b), np.ones(b), np.full(b, t), 1, L.MC_F32)
        assert lib.mc_kv4_append(C.byref(cache), C.byref(new), stream) == L.MC_OK
        held, self_out = ints(np.full(b, t + 1)), torch.empty_like(q)
        a = L.Kv4AttentionArgs(q=q.data_ptr(), out=self_out.data_ptr(), q_start=self.rows.data_ptr(),
                               q_len=self.one.data_ptr(), kv_len=held.data_ptr(), q_rows=b, q_row_stride=D,
                               q_head_stride=DIM, out_row_stride=D, out_head_stride=DIM, dtype=L.MC_F32, heads=HEADS,
                               max_q_len=1, max_kv_len=STEPS, causal=1, scale=DIM ** -0.5)
        assert lib.mc_kv4_attention_workspace(C.byref(cache), C.byref(a)) == 0
        assert lib.mc_kv4_attention(C.byref(cache), C.byref(a), stream) == L.MC_OK
        y = x + self_out.view(b, D) @ self.w["o"]
        cq = (y @ self.w["cq"]).view(b, HEADS, DIM).contiguous()
        cross_out = torch.empty_like(cq)
        ca, _ = cross_arguments(cq, self.enc_k, self.enc_v, cross_out, None, [self.rows, self.one] + self.source, None,
                                "f32", DIM ** -0.5, 1, int(self.k_len.max()))
        assert lib.mc_cross_attention(C.byref(ca), stream) == L.MC_OK
        logits = (y + cross_out.view(b, D)) @ self.out
        nxt, probs = torch.empty(b, dtype=torch.int32, device="cuda"), torch.empty(b, device="cuda")
        top_k, top_p = ints(np.full(b, 40)), torch.full((b,), 0.95, device="cuda")
        s = L.SampleArgs(logits=logits.data_ptr(), temperature=self.temperature.data_ptr(), top_k=top_k.data_ptr(),
                         top_p=top_p.data_ptr(), uniform=self.uniform[t].data_ptr(), tokens=nxt.data_ptr(),
                         probs=probs.data_ptr(), row_stride=VOCAB, dtype=L.MC_F32, rows=b, vocab=VOCAB)
        assert lib.mc_sample(C.byref(s), stream) == L.MC_OK
        torch.cuda.current_stream().synchronize()
        return dict(q=q, k=k, v=v, self_out=self_out, cq=cq, cross_out=cross_out, logits=logits, tokens=nxt, probs=probs)


@pytest.mark.parametrize("src_len,copies", [([17], 1), ([5, 40, 1], 3), ([64, 130], 40)])
def test_sampled_translations_step_by_step(src_len, copies):
    dec = Decoder(src_len, copies, seed=len(src_len) + copies)
    scale = DIM ** -0.5
    tokens = torch.arange(dec.batch, dtype=torch.int32, device="cuda") % VOCAB
    held = [[], []]
    enc_k, enc_v = f64(dec.enc_k), f64(dec.enc_v)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for t in range(STEPS):
            r = dec.step(t, tokens, stream.cuda_stream)
            for h, n in zip(held, ("k", "v")):
                c, s, m = quantize(f64(r[n]))
                h.append(m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * c)
            q, cq, got, cross = (f64(r[n]) for n in ("q", "cq", "self_out", "cross_out"))
            for i in range(dec.batch):
                k, v = (np.stack([row[i] for row in h]) for h in held)
                want, _ = kv_attend(q[i:i + 1], k, v, scale, lambda _: t + 1)
                tol = (2.0 ** -18 + 2 * score_error(q[i:i + 1], k, scale)) * np.abs(v).max()
                np.testing.assert_allclose(got[i:i + 1], want, rtol=0, atol=tol)
                at = slice(dec.k_start[i], dec.k_start[i] + dec.k_len[i])
                want, _ = cross_attend(cq[i:i + 1], enc_k[at], enc_v[at], scale, np.ones(dec.k_len[i], bool))
                dx = 2.0 ** -20 * scale * np.abs(cq[i]).sum(-1).max() * np.abs(enc_k[at]).max()
                np.testing.assert_allclose(cross[i:i + 1], want, rtol=0, atol=(2.0 ** -18 + 2 * dx) * np.abs(enc_v[at]).max())
            logits, u, temperature = f64(r["logits"]), f64(dec.uniform[t]), f64(dec.temperature)
            for i in range(dec.batch):
                token, prob = sample_reference(logits[i], temperature[i], 40, float(np.float32(0.95)), 0.0, u[i])
                assert int(r["tokens"][i]) == token and float(r["probs"][i]) == pytest.approx(prob, rel=2.0 ** -20)
            tokens = r["tokens"]
    assert status_bits() == 0
    if copies > 1:   # the copies of a source draw different translations
        assert len({int(x) for x in tokens}) > 1


def test_host_memory_is_refused_wherever_it_is_given():
    # every pointer but the one in question is good; nothing is launched
    lib = L.load()
    host = torch.zeros(4096, dtype=torch.uint8)
    at = (host.data_ptr() + 15) // 16 * 16
    room = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    base = room.data_ptr()
    zeros = room[:64].data_ptr()

    def refused(call, struct, fields):
        for f in fields:
            keep = getattr(struct, f)
            setattr(struct, f, at)
            assert call() == L.MC_INVALID_INPUT, f
            setattr(struct, f, keep)
        assert call() == L.MC_OK

    cache = L.Kv4Cache(pages=base, page_table=zeros, n_pages=4, page_tokens=16, kv_heads=1, head_dim=64, batch=1,
                       pages_per_seq=2)
    rows = L.Kv4Rows(k=base + 65536, v=base + 131072, start=zeros, count=zeros, first=zeros, rows=8, k_row_stride=64,
                     k_head_stride=64, v_row_stride=64, v_head_stride=64, dtype=L.MC_F32, max_count=4)
    for fn in (lib.mc_kv4_append, lib.mc_kv4_read):
        refused(lambda: fn(C.byref(cache), C.byref(rows), None), rows, ["k", "v", "start", "count", "first"])
        refused(lambda: fn(C.byref(cache), C.byref(rows), None), cache, ["pages", "page_table"])
    att = L.Kv4AttentionArgs(q=base + 65536, out=base + 131072, lse=base + 4096, q_start=zeros, q_len=zeros,
                             kv_len=zeros, q_rows=8, q_row_stride=64, q_head_stride=64, out_row_stride=64,
                             out_head_stride=64, dtype=L.MC_F32, heads=1, max_q_len=1, max_kv_len=32, scale=1.0)
    refused(lambda: lib.mc_kv4_attention(C.byref(cache), C.byref(att), None), att,
            ["q", "out", "lse", "q_start", "q_len", "kv_len"])
    cross = L.CrossAttentionArgs(q=base + 65536, k=base + 131072, v=base + 196608, out=base + 262144, lse=base + 4096,
                                 q_start=zeros, q_len=zeros, k_start=zeros, k_len=zeros, key_mask=zeros, q_rows=8,
                                 k_rows=8, q_row_stride=64, q_head_stride=64, k_row_stride=64, k_head_stride=64,
                                 v_row_stride=64, v_head_stride=64, out_row_stride=64, out_head_stride=64,
                                 dtype=L.MC_F32, batch=1, heads=1, kv_heads=1, head_dim=64, max_q_len=1, max_k_len=8,
                                 scale=1.0)
    refused(lambda: lib.mc_cross_attention(C.byref(cross), None), cross,
            ["q", "k", "v", "out", "lse", "q_start", "q_len", "k_start", "k_len", "key_mask"])
    draw = L.SampleArgs(logits=base + 65536, temperature=zeros, top_k=zeros, top_p=zeros, min_p=zeros, uniform=zeros,
                        tokens=base + 8192, probs=base + 12288, row_stride=100, dtype=L.MC_F32, rows=1, vocab=100)
    refused(lambda: lib.mc_sample(C.byref(draw), None), draw,
            ["logits", "temperature", "top_k", "top_p", "min_p", "uniform", "candidates", "tokens", "probs"])
    torch.cuda.synchronize()
    assert status_bits() == 0


def documented_step():
    """The Python lines of INTEGRATION.md's section on these operators."""
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    section = text[text.index("### Decode-step operators"):]
    return section[section.index("```python\n") + len("```python\n"):].split("```")[0]


@pytest.mark.parametrize("batch", [1, 3, 27, 28, 64])
def test_the_documented_step(batch):
    g = torch.Generator(device="cuda")
    g.manual_seed(batch)
    rng = np.random.default_rng(batch)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    held = Cache(batch, 16, 16, 8, 64, fill=0xFF)
    cs, lib, lens = held.struct(), L.load(), rng.integers(0, 255, batch)
    past = [rnd(int(lens.sum()) + 1, 8, 64) for _ in range(2)]
    before = rows_struct(*past, np.cumsum(lens) - lens, lens, np.zeros(batch), 255, L.MC_F32)
    assert lib.mc_kv4_append(C.byref(cs), C.byref(before), torch.cuda.current_stream().cuda_stream) == L.MC_OK
    src_len = rng.integers(1, 257, batch)
    src_start = np.cumsum(src_len) - src_len
    names = dict(
        batch=batch, pages=held.pages, table=held.table_dev, n_pages=held.n_pages, k=rnd(batch, 8, 64), v=rnd(batch, 8, 64),
        row=ints(np.arange(batch)), ones=ints(np.ones(batch)), length=ints(lens), length_plus_1=ints(lens + 1),
        q=rnd(batch, 8, 64), out=torch.zeros(batch, 8, 64, device="cuda"), cq=rnd(batch, 8, 64),
        co=torch.zeros(batch, 8, 64, device="cuda"), enc_k=rnd(int(src_len.sum()), 8, 64),
        enc_v=rnd(int(src_len.sum()), 8, 64), src_start=ints(src_start), src_len=ints(src_len),
        logits=rnd(batch, 32000) * 2, temperature=torch.full((batch,), 0.8, device="cuda"),
        top_p=torch.full((batch,), 0.9, device="cuda"), uniform=torch.rand(batch, generator=g, device="cuda"),
        tokens=torch.full((batch,), -7, dtype=torch.int32, device="cuda"), stream=torch.cuda.current_stream().cuda_stream)
    exec(compile(documented_step(), "INTEGRATION.md", "exec"), names)
    torch.cuda.synchronize()
    assert status_bits() == 0
    back = [torch.zeros(int(lens.sum()) + batch, 8, 64, device="cuda") for _ in range(2)]
    total = lens + 1
    at = np.cumsum(total) - total
    read = rows_struct(*back, at, total, np.zeros(batch), 256, L.MC_F32)
    assert lib.mc_kv4_read(C.byref(cs), C.byref(read), names["stream"]) == L.MC_OK
    torch.cuda.synchronize()
    q, out, cq, co, enc_k, enc_v = (f64(names[n]) for n in ("q", "out", "cq", "co", "enc_k", "enc_v"))
    k, v = (f64(x) for x in back)
    for i in range(batch):
        ki, vi = k[at[i]:at[i] + total[i]], v[at[i]:at[i] + total[i]]
        want, _ = kv_attend(q[i:i + 1], ki, vi, 0.125, lambda _: total[i])
        tol = (2.0 ** -18 + 2 * score_error(q[i:i + 1], ki, 0.125)) * np.abs(vi).max()
        np.testing.assert_allclose(out[i:i + 1], want, rtol=0, atol=tol)
        src = slice(src_start[i], src_start[i] + src_len[i])
        want, _ = cross_attend(cq[i:i + 1], enc_k[src], enc_v[src], 0.125, np.ones(src_len[i], bool))
        dx = 2.0 ** -20 * 0.125 * np.abs(cq[i]).sum(-1).max() * np.abs(enc_k[src]).max()
        np.testing.assert_allclose(co[i:i + 1], want, rtol=0, atol=(2.0 ** -18 + 2 * dx) * np.abs(enc_v[src]).max())
        token, _ = sample_reference(f64(names["logits"])[i], float(np.float32(0.8)), 0, float(np.float32(0.9)), 0.0,
                                    float(f64(names["uniform"])[i]))
        assert int(names["tokens"][i]) == token


@pytest.mark.parametrize("code", [L.MC_F32, L.MC_BF16])
@pytest.mark.parametrize("q_len", [1, 200])
def test_tensors_of_no_rows_may_be_null(code, q_len):
    # no keys at all, no queries, no new rows, no pages: nothing is read, and a length that says otherwise
    # is reported
    lib, stream = L.load(), torch.cuda.current_stream().cuda_stream
    dtype = torch.float32 if code == L.MC_F32 else torch.bfloat16
    zero, one, full = ints([0, 0]), ints([1, 1]), ints([q_len, 0])
    q, out, lse = torch.ones(q_len, 2, 64, dtype=dtype, device="cuda"), torch.full((q_len, 2, 64), 7.0, dtype=dtype, device="cuda"), torch.zeros(q_len, 2, device="cuda")
    strides = dict(q_row_stride=128, q_head_stride=64, out_row_stride=128, out_head_stride=64)
    rows = dict(q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), q_start=zero.data_ptr(), q_len=full.data_ptr())
    room = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    kv = dict(k_row_stride=128, k_head_stride=64, v_row_stride=128, v_head_stride=64)
    cross = L.CrossAttentionArgs(**rows, **strides, **kv, k_start=zero.data_ptr(), k_len=zero.data_ptr(), q_rows=q_len, k_rows=0,
                                 workspace=room.data_ptr(), workspace_bytes=1 << 24, dtype=code, batch=2, heads=2,
                                 kv_heads=2, head_dim=64, max_q_len=q_len, max_k_len=300, scale=0.125)
    assert lib.mc_cross_attention(C.byref(cross), stream) == L.MC_OK and status_bits() == 0
    assert bool((out == 0).all()) and bool(lse.isneginf().all())
    cross.k_len = one.data_ptr()      # both sequences say that they have a key
    out.fill_(7.0)
    assert lib.mc_cross_attention(C.byref(cross), stream) == L.MC_OK and status_bits() == 4
    assert bool((out == 7).all())
    table = ints([0, 0])
    cache = L.Kv4Cache(page_table=table.data_ptr(), n_pages=0, page_tokens=16, kv_heads=2, head_dim=64, batch=2, pages_per_seq=1)
    att = L.Kv4AttentionArgs(**rows, **strides, kv_len=zero.data_ptr(), q_rows=q_len, workspace=room.data_ptr(),
                             workspace_bytes=1 << 24, dtype=code, heads=2, max_q_len=q_len, max_kv_len=16, scale=0.125)
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), stream) == L.MC_OK and status_bits() == 0
    assert bool((out == 0).all()) and bool(lse.isneginf().all())
    att.kv_len = one.data_ptr()       # a page that is not there
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), stream) == L.MC_OK and status_bits() == 4
    new = L.Kv4Rows(start=zero.data_ptr(), count=zero.data_ptr(), first=zero.data_ptr(), rows=0, **kv, dtype=code, max_count=3)
    for fn in (lib.mc_kv4_append, lib.mc_kv4_read):
        new.count = zero.data_ptr()
        assert fn(C.byref(cache), C.byref(new), stream) == L.MC_OK and status_bits() == 0
        new.count = one.data_ptr()
        assert fn(C.byref(cache), C.byref(new), stream) == L.MC_OK and status_bits() == 4
    att.q_rows, att.q, att.out, att.lse, att.kv_len = 0, None, None, None, zero.data_ptr()
    cross.q_rows, cross.q, cross.out, cross.lse, cross.k_len = 0, None, None, None, zero.data_ptr()
    for lens, bits in ((zero, 0), (one, 4)):
        att.q_len = cross.q_len = lens.data_ptr()
        assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), stream) == L.MC_OK and status_bits() == bits
        assert lib.mc_cross_attention(C.byref(cross), stream) == L.MC_OK and status_bits() == bits
    for struct, field in ((cross, "k_rows"), (cross, "q_rows"), (att, "q_rows")):
        setattr(struct, field, 1)
        assert (lib.mc_cross_attention(C.byref(struct), stream) if struct is cross else
                lib.mc_kv4_attention(C.byref(cache), C.byref(struct), stream)) == L.MC_INVALID_INPUT
        setattr(struct, field, 0)
