"""The 4-bit cache (mc_kv4_append / mc_kv4_read / mc_kv4_attention) against
plain 64-bit forms of its definition, at page borders, odd head sizes, empty
rows, stale page contents and bad indexes.

Tolerances, derived from the arithmetic.  Quantizing is exact, so codes and
read-back values are compared bit for bit.  Attention works on row = minimum +
scale * code, whose parts are at most 3 max|row| together.  A score is a sum
of q times those parts with 22 bits in each product (f32; 16-bit q is exact)
and f32 sums: it is within dx = 2^-21 * attention scale * sum|q| * 3 max|k| of
its value, which moves an output by at most 2 dx max|v|.  The weights meet the
values rounded to 11 bits (16-bit types: 2^-12 each way, on parts of up to
3 max|v|, independent of one another) or to 22 (f32), sums over up to 2^12 keys
lose at most 2^-19 more, and the output is rounded once (eps / 2).  So
f32: (2^-18 + 2 dx) max|v|, 16 bits: (eps / 2 + 2^-11 + 2 dx) max|v|; and as the
f32 errors are independent, their root mean square is far less: 2^-19 max|v|.
"""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from marian_cuda import _lib as L  # noqa: E402

gpu = pytest.mark.gpu
DTYPES = {"f32": (torch.float32, L.MC_F32), "f16": (torch.float16, L.MC_F16), "bf16": (torch.bfloat16, L.MC_BF16)}


# ---- the definition, in 64 bits -------------------------------------------------

def quantize(x):
    """x [..., d] float64 holding the typed inputs -> codes, scale, minimum (float64 of the stored float16)."""
    x = x.astype(np.float64)
    minimum = x.min(-1).astype(np.float32).astype(np.float16)
    span = (x.max(-1).astype(np.float32) - minimum.astype(np.float32)).astype(np.float32)
    scale = (span * np.float32(1.0 / 15.0)).astype(np.float16)
    s, m = scale.astype(np.float64)[..., None], minimum.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.clip(np.rint((x - m) / s), 0, 15), 0.0)
    return c, scale, minimum


def pack_pages(codes, scale, minimum, pages, table, t, d):
    """Writes codes [2, b, n, hk, d] and pairs into pages (numpy uint8 [n_pages, hk, t * (d + 8)])."""
    _, b, n, hk, _ = codes.shape
    c = codes.astype(np.uint8)
    packed = c[..., 0::2] | (c[..., 1::2] << 4)
    pairs = np.stack([scale, minimum], -1).astype(np.float16)
    for w in range(2):
        for i in range(b):
            for p in range(n):
                block = pages[table[i, p // t]]
                s = p % t
                block[:, (w * t + s) * (d // 2):(w * t + s + 1) * (d // 2)] = packed[w, i, p]
                at = t * d + (w * t + s) * 4
                block[:, at:at + 4] = np.ascontiguousarray(pairs[w, i, p]).view(np.uint8).reshape(hk, 4)


def attend(q, k, v, scale, q0_limit):
    """One sequence: q [m, h, d], k, v [n, hk, d] -> out [m, h, d], lse [m, h]; query i sees keys below q0_limit(i)."""
    m, h, d = q.shape
    group = h // k.shape[1]
    out, lse = np.zeros((m, h, d)), np.full((m, h), -np.inf)
    for i in range(m):
        n = max(0, q0_limit(i))
        if n == 0:
            continue
        for j in range(h):
            x = (k[:n, j // group] @ q[i, j]) * scale
            top = x.max()
            w = np.exp(x - top)
            out[i, j] = w @ v[:n, j // group] / w.sum()
            lse[i, j] = top + math.log(w.sum())
    return out, lse


# ---- calls ------------------------------------------------------------------------

class Cache:
    def __init__(self, b, per_seq, t, hk, d, extra=3, seed=0, fill=0xA5):
        rng = np.random.default_rng(seed)
        self.t, self.hk, self.d, self.b, self.per_seq = t, hk, d, b, per_seq
        self.n_pages = b * per_seq + extra
        self.table = rng.permutation(self.n_pages)[:b * per_seq].reshape(b, per_seq).astype(np.int32)
        # every byte 0xFF: codes 15 and NaN pairs where nothing has been written
        self.pages = torch.full((self.n_pages, hk, t * (d + 8)), fill, dtype=torch.uint8, device="cuda")
        self.table_dev = torch.from_numpy(self.table).cuda()

    def struct(self):
        return L.Kv4Cache(pages=self.pages.data_ptr(), page_table=self.table_dev.data_ptr(), n_pages=self.n_pages,
                          page_tokens=self.t, kv_heads=self.hk, head_dim=self.d, batch=self.b,
                          pages_per_seq=self.per_seq)


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def rows_struct(k, v, start, count, first, max_count, code):
    keep = [k, v, ints(start), ints(count), ints(first)]
    s = L.Kv4Rows(k=k.data_ptr(), v=v.data_ptr(), start=keep[2].data_ptr(), count=keep[3].data_ptr(),
                  first=keep[4].data_ptr(), rows=k.shape[0], k_row_stride=k.stride(0), k_head_stride=k.stride(1),
                  v_row_stride=v.stride(0), v_head_stride=v.stride(1), dtype=code, max_count=max_count)
    s.keep = keep
    return s


def status_bits():
    bits = C.c_uint32(0)
    assert L.load().mc_op_status(C.byref(bits)) == L.MC_OK
    return bits.value


def call(fn, *structs):
    torch.cuda.synchronize()
    return fn(*[C.byref(s) for s in structs], torch.cuda.current_stream().cuda_stream)


def attention(cache, q, q_start, q_len, kv_len, scale, causal, dtype, max_q=None, max_kv=None, out=None, stream=None):
    lib = L.load()
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    keep = [ints(q_start), ints(q_len), ints(kv_len)]
    a = L.Kv4AttentionArgs(q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), q_start=keep[0].data_ptr(),
                           q_len=keep[1].data_ptr(), kv_len=keep[2].data_ptr(), q_rows=q.shape[0],
                           q_row_stride=q.stride(0), q_head_stride=q.stride(1), out_row_stride=out.stride(0),
                           out_head_stride=out.stride(1), dtype=DTYPES[dtype][1], heads=q.shape[1],
                           max_q_len=int(max(q_len)) if max_q is None else max_q,
                           max_kv_len=int(max(kv_len)) if max_kv is None else max_kv, causal=causal, scale=scale)
    c = cache.struct()
    need = lib.mc_kv4_attention_workspace(C.byref(c), C.byref(a))
    ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    torch.cuda.synchronize()
    assert lib.mc_kv4_attention(C.byref(c), C.byref(a), torch.cuda.current_stream().cuda_stream) == L.MC_OK
    torch.cuda.synchronize()
    return out, lse, need


def typed(rng, shape, dtype, size=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * size).astype(np.float32)).to(DTYPES[dtype][0])


def f64(x):
    return x.float().cpu().numpy().astype(np.float64)


# ---- refusals: no GPU needed ----------------------------------------------------

def host_args():
    cache = L.Kv4Cache(pages=1 << 20, page_table=1 << 20, n_pages=8, page_tokens=16, kv_heads=2, head_dim=64, batch=2,
                       pages_per_seq=4)
    rows = L.Kv4Rows(k=1 << 20, v=1 << 21, start=64, count=64, first=64, rows=10, k_row_stride=128, k_head_stride=64,
                     v_row_stride=128, v_head_stride=64, dtype=L.MC_BF16, max_count=5)
    att = L.Kv4AttentionArgs(q=1 << 20, out=1 << 21, lse=64, q_start=64, q_len=64, kv_len=64, workspace=1 << 20,
                             workspace_bytes=1 << 40, q_rows=10, q_row_stride=256, q_head_stride=64,
                             out_row_stride=256, out_head_stride=64, dtype=L.MC_F32, heads=4, max_q_len=3,
                             max_kv_len=60, causal=1, scale=0.125)
    return cache, rows, att


CACHE_FAULTS = [("page_tokens", 12), ("page_tokens", 64), ("page_tokens", 0), ("head_dim", 40), ("head_dim", 144),
                ("head_dim", 0), ("kv_heads", 0), ("batch", -1), ("pages_per_seq", 0), ("pages_per_seq", 1 << 30),
                ("n_pages", -1), ("pages", 0), ("pages", (1 << 20) + 8), ("page_table", 0), ("page_table", 6)]


@pytest.mark.parametrize("field,value", CACHE_FAULTS)
def test_bad_caches_are_refused(field, value):
    lib = L.load()
    cache, rows, att = host_args()
    setattr(cache, field, value)
    for fn, arg in ((lib.mc_kv4_append, rows), (lib.mc_kv4_read, rows), (lib.mc_kv4_attention, att)):
        assert fn(C.byref(cache), C.byref(arg), None) == L.MC_INVALID_INPUT


@pytest.mark.parametrize("field,value", [("k", 0), ("v", (1 << 21) + 4), ("start", 0), ("count", 0), ("first", 2),
                                         ("rows", -1), ("k_row_stride", 12), ("k_row_stride", -128),
                                         ("v_head_stride", 4), ("dtype", 3), ("dtype", -1), ("max_count", -1)])
def test_bad_rows_are_refused(field, value):
    lib = L.load()
    cache, rows, _ = host_args()
    setattr(rows, field, value)
    for fn in (lib.mc_kv4_append, lib.mc_kv4_read):
        assert fn(C.byref(cache), C.byref(rows), None) == L.MC_INVALID_INPUT


def test_overlapping_output_rows_are_refused():
    lib = L.load()
    for field, value in (("k_head_stride", 48), ("v_row_stride", 64), ("k_row_stride", 0)):
        cache, rows, _ = host_args()
        setattr(rows, field, value)
        assert lib.mc_kv4_read(C.byref(cache), C.byref(rows), None) == L.MC_INVALID_INPUT
    cache, rows, _ = host_args()
    rows.v = rows.k
    assert lib.mc_kv4_read(C.byref(cache), C.byref(rows), None) == L.MC_INVALID_INPUT


@pytest.mark.parametrize("field,value", [("q", 0), ("out", 0), ("out", 1 << 20), ("out", (1 << 21) + 8), ("lse", 6),
                                         ("q_start", 0), ("q_len", 0), ("kv_len", 0), ("q_rows", -1),
                                         ("q_row_stride", 255), ("out_head_stride", 32), ("out_row_stride", 128),
                                         ("dtype", 7), ("heads", 3), ("heads", 0), ("max_q_len", -1),
                                         ("max_kv_len", -1), ("max_kv_len", 65), ("scale", float("nan")),
                                         ("scale", float("inf"))])
def test_bad_attention_arguments_are_refused(field, value):
    lib = L.load()
    cache, _, att = host_args()
    setattr(att, field, value)
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_INVALID_INPUT


def test_short_workspace_is_refused():
    lib = L.load()
    cache, _, att = host_args()
    cache.batch, cache.pages_per_seq, att.max_q_len, att.max_kv_len = 1, 4096, 1, 60000
    need = lib.mc_kv4_attention_workspace(C.byref(cache), C.byref(att))
    assert need > 0
    for ws, n in ((0, need), (1 << 20, need - 1), ((1 << 20) + 8, need)):
        att.workspace, att.workspace_bytes = ws, n
        assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_INVALID_INPUT


def test_null_structs_and_empty_calls():
    lib = L.load()
    cache, rows, att = host_args()
    assert lib.mc_kv4_append(None, C.byref(rows), None) == L.MC_INVALID_INPUT
    assert lib.mc_kv4_append(C.byref(cache), None, None) == L.MC_INVALID_INPUT
    assert lib.mc_kv4_attention(C.byref(cache), None, None) == L.MC_INVALID_INPUT
    assert lib.mc_kv4_attention_workspace(None, None) == 0
    cache.batch = 0
    assert lib.mc_kv4_append(C.byref(cache), C.byref(rows), None) == L.MC_OK
    assert lib.mc_kv4_read(C.byref(cache), C.byref(rows), None) == L.MC_OK
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_OK
    cache.batch, rows.max_count, att.max_q_len = 2, 0, 0
    assert lib.mc_kv4_append(C.byref(cache), C.byref(rows), None) == L.MC_OK
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is present")
def test_sound_arguments_need_a_device():
    lib = L.load()
    cache, rows, att = host_args()
    assert lib.mc_kv4_append(C.byref(cache), C.byref(rows), None) == L.MC_CUDA
    assert lib.mc_kv4_read(C.byref(cache), C.byref(rows), None) == L.MC_CUDA
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_CUDA


def test_page_bytes():
    lib = L.load()
    assert lib.mc_kv4_page_bytes(16, 8, 64) == 8 * 16 * (2 * 32 + 8)
    assert lib.mc_kv4_page_bytes(8, 1, 16) == 8 * 24
    assert lib.mc_kv4_page_bytes(10, 1, 16) == 0 and lib.mc_kv4_page_bytes(16, 0, 64) == 0


# ---- rows in and out -----------------------------------------------------------

@gpu
def test_host_memory_is_refused():
    lib = L.load()
    cache, rows, att = host_args()
    host = torch.zeros(1 << 16, dtype=torch.uint8)
    at = (host.data_ptr() + 15) // 16 * 16
    cache.pages = at
    assert lib.mc_kv4_append(C.byref(cache), C.byref(rows), None) == L.MC_INVALID_INPUT
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_INVALID_INPUT


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,t,hk,counts,firsts", [
    (64, 16, 8, [1, 0, 1, 1], [0, 5, 31, 47]), (48, 8, 3, [17, 1, 40], [3, 8, 0]), (128, 32, 2, [70], [29]),
    (16, 16, 1, [5, 33], [11, 0]), (80, 8, 2, [9, 2], [7, 15]), (112, 16, 1, [3], [14]), (32, 32, 5, [33, 32], [0, 31])])
def test_rows_are_quantized_by_the_definition(dtype, d, t, hk, counts, firsts):
    lib, rng = L.load(), np.random.default_rng(d + t)
    b = len(counts)
    per_seq = -(-max(f + n for f, n in zip(firsts, counts)) // t)
    cache = Cache(b, per_seq, t, hk, d, fill=0xFF)
    start = np.cumsum(counts) - counts + 2
    rows = int(np.sum(counts)) + 3
    k, v = typed(rng, (rows, hk, d), dtype), typed(rng, (rows, hk, d), dtype, 3.0)
    k[start[0]] = 0.25          # a constant row: scale 0
    v[start[0], 0, :4] = torch.tensor([0.5, -0.5, 1.5, 7.5]).to(v.dtype)
    # steps of exactly 1 from 0 to 15: the halves between are ties
    ties = torch.arange(d, dtype=torch.float32) % 31 / 2
    ties[:2] = torch.tensor([0.0, 15.0])
    k[start[0] + counts[0] - 1, hk - 1] = ties.to(k.dtype)
    want = cache.pages.cpu().numpy()
    for w, x in ((0, k), (1, v)):
        c, s, m = quantize(f64(x))
        for i in range(b):
            for j in range(counts[i]):
                p, r = firsts[i] + j, start[i] + j
                block, slot = want[cache.table[i, p // t]], p % t
                u = c[r].astype(np.uint8)
                block[:, (w * t + slot) * (d // 2):(w * t + slot + 1) * (d // 2)] = u[:, 0::2] | (u[:, 1::2] << 4)
                at = t * d + (w * t + slot) * 4
                block[:, at:at + 4] = np.ascontiguousarray(np.stack([s[r], m[r]], -1)).view(np.uint8).reshape(hk, 4)
    rs = rows_struct(k.cuda(), v.cuda(), start, counts, firsts, max(counts), DTYPES[dtype][1])
    cs = cache.struct()
    assert call(lib.mc_kv4_append, cs, rs) == L.MC_OK
    assert status_bits() == 0
    np.testing.assert_array_equal(cache.pages.cpu().numpy(), want)  # every other byte as it was

    back = [torch.full((rows, hk, d), 9.0, dtype=k.dtype, device="cuda") for _ in range(2)]
    rb = rows_struct(*back, start, counts, firsts, max(counts), DTYPES[dtype][1])
    assert call(lib.mc_kv4_read, cs, rb) == L.MC_OK
    assert status_bits() == 0
    live = np.zeros(rows, bool)
    for i in range(b):
        live[start[i]:start[i] + counts[i]] = True
    for x, got in zip((k, v), back):
        c, s, m = quantize(f64(x))
        value = (m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * c).astype(np.float32)
        value = torch.from_numpy(value).to(k.dtype)
        got = got.cpu()
        assert torch.equal(got[live], value[live])
        assert torch.equal(got[~live], torch.full_like(got[~live], 9.0))


@gpu
def test_near_ties_round_as_the_real_quotient():
    # minimum 0, scale 1 (maximum 15): codes of c + 1/2 exactly, and of its two
    # neighbours in f32, where a single-precision quotient cannot be trusted
    lib = L.load()
    d, t = 128, 16
    halves = np.arange(15) + 0.5
    x = np.zeros((1, 1, d), np.float32)
    x[0, 0, 1] = 15.0
    x[0, 0, 2:17] = halves
    x[0, 0, 17:32] = np.nextafter(halves.astype(np.float32), np.float32(0))
    x[0, 0, 32:47] = np.nextafter(halves.astype(np.float32), np.float32(100))
    y = x * np.float32(1 / 3) + np.float32(0.7)  # a scale that is not a power of two
    cache = Cache(1, 1, t, 1, d)
    rs = rows_struct(torch.from_numpy(x).cuda(), torch.from_numpy(y).cuda(), [0], [1], [0], 1, L.MC_F32)
    cs = cache.struct()
    assert call(lib.mc_kv4_append, cs, rs) == L.MC_OK
    page = cache.pages.cpu().numpy()[cache.table[0, 0], 0]
    for w, z in ((0, x), (1, y)):
        c, _, _ = quantize(z.astype(np.float64))
        got = page[w * t * d // 2:w * t * d // 2 + d // 2]
        np.testing.assert_array_equal(np.stack([got & 15, got >> 4], -1).reshape(-1), c[0, 0])


@gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 1e6, -1e6])
def test_rows_that_cannot_be_held_are_zeros_and_reported(bad):
    lib = L.load()
    cache = Cache(1, 1, 8, 2, 32)
    k = torch.randn(3, 2, 32, device="cuda")
    k[1, 1, 31] = bad
    rs = rows_struct(k, torch.randn(3, 2, 32, device="cuda"), [0], [3], [2], 3, L.MC_F32)
    cs = cache.struct()
    assert call(lib.mc_kv4_append, cs, rs) == L.MC_OK
    assert status_bits() == 1
    back = [torch.empty(3, 2, 32, device="cuda") for _ in range(2)]
    rb = rows_struct(*back, [0], [3], [2], 3, L.MC_F32)
    assert call(lib.mc_kv4_read, cs, rb) == L.MC_OK and status_bits() == 0
    assert bool((back[0][1, 1] == 0).all()) and bool((back[0][1, 0] != 0).any()) and bool(torch.isfinite(back[0]).all())


@gpu
def test_strided_and_head_major_rows():
    lib, rng = L.load(), np.random.default_rng(5)
    d, t, hk, n = 64, 16, 4, 21
    qkv = typed(rng, (n, 3, hk, d), "bf16").cuda()      # interleaved projections
    k, v = qkv[:, 1], typed(rng, (hk, n, d), "bf16").cuda().transpose(0, 1)   # [hk, n, d] storage
    cache, plain = Cache(1, 2, t, hk, d, seed=1), Cache(1, 2, t, hk, d, seed=1)
    for c, (x, y) in ((cache, (k, v)), (plain, (k.contiguous(), v.contiguous()))):
        cs, rs = c.struct(), rows_struct(x, y, [0], [n], [4], n, L.MC_BF16)
        assert call(lib.mc_kv4_append, cs, rs) == L.MC_OK
    assert torch.equal(cache.pages, plain.pages)
    back = torch.zeros(hk, n, d, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    wide = torch.zeros(n, 2, hk, d, dtype=torch.bfloat16, device="cuda")
    dense = [torch.zeros(n, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cs = cache.struct()
    assert call(lib.mc_kv4_read, cs, rows_struct(back, wide[:, 1], [0], [n], [4], n, L.MC_BF16)) == L.MC_OK
    assert call(lib.mc_kv4_read, cs, rows_struct(*dense, [0], [n], [4], n, L.MC_BF16)) == L.MC_OK
    assert torch.equal(back, dense[0]) and torch.equal(wide[:, 1], dense[1]) and bool((wide[:, 0] == 0).all())


@gpu
@pytest.mark.parametrize("field,values", [("start", [0, 9]), ("start", [0, -1]), ("count", [3, 6]), ("count", [3, -1]),
                                          ("first", [0, 30]), ("first", [0, -2]), ("first", [0, 2147483647])])
def test_rows_out_of_bounds_are_left_out_and_reported(field, values):
    lib = L.load()
    cache = Cache(2, 2, 16, 1, 32)
    before = cache.pages.clone()
    given = {"start": [0, 3], "count": [3, 3], "first": [0, 5], field: values}
    k = torch.randn(10, 1, 32, device="cuda")
    rs = rows_struct(k, k * 2, given["start"], given["count"], given["first"], 5, L.MC_F32)
    cs = cache.struct()
    assert call(lib.mc_kv4_append, cs, rs) == L.MC_OK
    assert status_bits() == 4
    assert torch.equal(cache.pages[cache.table[1].astype(np.int64)], before[cache.table[1].astype(np.int64)])
    assert not torch.equal(cache.pages[int(cache.table[0, 0])], before[int(cache.table[0, 0])])


@gpu
def test_bad_page_ids_are_left_out_and_reported():
    lib, rng = L.load(), np.random.default_rng(3)
    t, hk, d, h = 8, 2, 64, 4
    cache = Cache(1, 5, t, hk, d)
    k, v = typed(rng, (40, hk, d), "f32"), typed(rng, (40, hk, d), "f32")
    cs = cache.struct()
    assert call(lib.mc_kv4_append, cs, rows_struct(k.cuda(), v.cuda(), [0], [40], [0], 40, L.MC_F32)) == L.MC_OK
    assert status_bits() == 0
    kc, ks, km = quantize(f64(k))
    vc, vs, vm = quantize(f64(v))
    keep = np.r_[0:8, 16:24, 32:37]    # pages 1 and 3 are bad
    kd = (km.astype(float)[..., None] + ks.astype(float)[..., None] * kc)[keep]
    vd = (vm.astype(float)[..., None] + vs.astype(float)[..., None] * vc)[keep]
    for bad in (-1, cache.n_pages, 2147483647):
        table = cache.table.copy()
        table[0, [1, 3]] = bad
        cache.table_dev = torch.from_numpy(table).cuda()
        q = typed(rng, (1, h, d), "f32")
        out, lse, _ = attention(cache, q.cuda(), [0], [1], [37], 0.125, 0, "f32")
        assert status_bits() == 4
        want, wl = attend(f64(q), kd, vd, 0.125, lambda i: len(keep))
        dx = score_error(f64(q), kd, 0.125)
        np.testing.assert_allclose(f64(out), want, atol=(2.0 ** -18 + 2 * dx) * np.abs(vd).max())
        np.testing.assert_allclose(f64(lse), wl, atol=2.0 ** -19 + dx)
        back = [torch.full((40, hk, d), 9.0, device="cuda") for _ in range(2)]
        cs = cache.struct()
        assert call(lib.mc_kv4_read, cs, rows_struct(*back, [0], [40], [0], 40, L.MC_F32)) == L.MC_OK
        assert status_bits() == 4
        assert bool((back[0][8:16] == 9).all()) and bool((back[1][0:8] != 9).any())


# ---- attention -------------------------------------------------------------------

def filled(rng, cache, lens, dtype="f32", k_shift=0.0):
    """A cache whose sequences hold lens[i] rows; the values they stand for, [b][n, hk, d] each."""
    lib = L.load()
    b, hk, d = cache.b, cache.hk, cache.d
    start = np.cumsum(lens) - lens
    k = typed(rng, (int(np.sum(lens)) + 1, hk, d), dtype) + k_shift
    v = typed(rng, (int(np.sum(lens)) + 1, hk, d), dtype)
    cs = cache.struct()
    rs = rows_struct(k.cuda(), v.cuda(), start, lens, np.zeros(b), max(1, int(max(lens))), DTYPES[dtype][1])
    assert call(lib.mc_kv4_append, cs, rs) == L.MC_OK and status_bits() == 0
    out = []
    for x in (k, v):
        c, s, m = quantize(f64(x))
        value = m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * c
        out.append([value[i0:i0 + n] for i0, n in zip(start, lens)])
    return out


def score_error(q, k, scale):
    """How far a score may be from its value: q [m, h, d], k [n, hk, d]."""
    return 2.0 ** -21 * scale * np.abs(q).sum(-1).max() * 3 * np.abs(k).max() if k.size else 0.0


def check(cache, rng, lens, q_lens, h, dtype, causal, gap=0, k_shift=0.0):
    ks, vs = filled(rng, cache, lens, k_shift=k_shift)
    d, scale = cache.d, cache.d ** -0.5
    q_start = np.cumsum(q_lens) - q_lens + gap * np.arange(len(q_lens))
    rows = int(np.sum(q_lens)) + gap * len(q_lens) + 1
    q = typed(rng, (rows, h, d), dtype)
    out, lse, need = attention(cache, q.cuda(), q_start, q_lens, lens, scale, causal, dtype,
                               max_kv=min(cache.per_seq * cache.t, max(1, max(lens))))
    assert status_bits() == 0
    eps = torch.finfo(q.dtype).eps
    touched = np.zeros(rows, bool)
    for i, (n, m) in enumerate(zip(lens, q_lens)):
        at = slice(q_start[i], q_start[i] + m)
        touched[at] = True
        if m == 0:
            continue
        want, wl = attend(f64(q)[at], ks[i], vs[i], scale, (lambda j: n - (m - 1 - j)) if causal else (lambda j: n))
        big = np.abs(vs[i]).max() if n else 1.0
        dx = score_error(f64(q)[at], ks[i], scale)
        tol = (2.0 ** -18 if dtype == "f32" else eps / 2 + 2.0 ** -11) + 2 * dx
        np.testing.assert_allclose(f64(out)[at], want, rtol=0, atol=tol * big)
        if dtype == "f32":
            assert np.sqrt(np.mean((f64(out)[at] - want) ** 2)) <= 2.0 ** -19 * big
        np.testing.assert_allclose(f64(lse)[at], wl, rtol=2.0 ** -20, atol=2.0 ** -19 + dx)
    assert bool((out[torch.from_numpy(~touched).cuda()] == 7).all()) and bool((lse[torch.from_numpy(~touched).cuda()] == 7).all())
    return need


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("t", [8, 16, 32])
def test_attention_of_single_tokens(dtype, d, t):
    rng = np.random.default_rng(d * t)
    lens = [1, 0, 31, 32, 33, t, t + 1, 130]
    cache = Cache(len(lens), -(-130 // t), t, 2, d, fill=0xFF)
    check(cache, rng, lens, [1] * len(lens), 2, dtype, 1)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("d,hk,group", [(64, 2, 1), (48, 1, 7), (128, 2, 4), (32, 1, 16), (96, 3, 3)])
def test_attention_of_chunks_with_shared_heads(dtype, causal, d, hk, group):
    rng = np.random.default_rng(d + group)
    lens, q_lens = [5, 70, 0, 33, 3], [5, 13, 2, 1, 6]   # more queries than keys, no keys, an odd rest
    cache = Cache(len(lens), 5, 16, hk, d, fill=0xFF)
    check(cache, rng, lens, q_lens, hk * group, dtype, causal, gap=2)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,hk,group,q_len", [([230], 8, 1, 1), ([2111], 1, 1, 1), ([3001, 40, 0], 1, 4, 1),
                                                ([1500, 1499], 2, 2, 5), ([700] * 3, 2, 1, 1)])
def test_attention_with_split_keys(dtype, lens, hk, group, q_len):
    rng = np.random.default_rng(len(lens) + hk)
    cache = Cache(len(lens), -(-max(lens) // 16), 16, hk, 64, fill=0xFF)
    check(cache, rng, lens, [q_len] * len(lens), hk * group, dtype, 1)


@gpu
def test_split_keys_are_used_and_agree_with_unsplit_ones():
    rng = np.random.default_rng(2)
    cache = Cache(1, 200, 16, 1, 64)
    assert check(cache, rng, [3190], [1], 1, "f32", 0) > 0
    assert check(Cache(64, 2, 16, 8, 64), rng, [32] * 64, [1] * 64, 8, "f32", 0) == 0


@gpu
@pytest.mark.parametrize("shift", [30.0, -200.0])
def test_attention_with_keys_far_from_zero(shift):
    # scores that all carry q . shift: the maximum has to follow them
    rng = np.random.default_rng(8)
    cache = Cache(2, 9, 16, 2, 64)
    ks, vs = filled(rng, cache, [140, 77], k_shift=shift)
    q = typed(rng, (2, 2, 64), "f32")
    out, lse, _ = attention(cache, q.cuda(), [0, 1], [1, 1], [140, 77], 0.125, 0, "f32")
    for i in range(2):
        want, wl = attend(f64(q)[i:i + 1], ks[i], vs[i], 0.125, lambda j: len(ks[i]))
        dx = score_error(f64(q)[i:i + 1], ks[i], 0.125)
        np.testing.assert_allclose(f64(out)[i:i + 1], want, atol=(2.0 ** -18 + 2 * dx) * np.abs(vs[i]).max())
        np.testing.assert_allclose(f64(lse)[i:i + 1], wl, rtol=2.0 ** -20, atol=2.0 ** -19 + dx)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_value_rows_of_very_different_sizes(dtype):
    # scales from 2^-20 to 2^9 and constant rows (scale 0) side by side
    lib, rng = L.load(), np.random.default_rng(11)
    cache = Cache(1, 3, 16, 1, 32)
    k, v = typed(rng, (45, 1, 32), "f32"), typed(rng, (45, 1, 32), "f32")
    v *= torch.from_numpy(2.0 ** rng.integers(-16, 10, (45, 1, 1)).astype(np.float32))
    v[7], v[20] = 3.0, 0.0
    cs = cache.struct()
    assert call(lib.mc_kv4_append, cs, rows_struct(k.cuda(), v.cuda(), [0], [45], [0], 45, L.MC_F32)) == L.MC_OK
    kd, vd = ((lambda c, s, m: m.astype(float)[..., None] + s.astype(float)[..., None] * c)(*quantize(f64(x))) for x in (k, v))
    for size in (1.0, 20.0):   # flat weights and nearly one-hot ones
        q = typed(rng, (1, 1, 32), dtype, size)
        out, _, _ = attention(cache, q.cuda(), [0], [1], [45], 32 ** -0.5, 0, dtype)
        want, _ = attend(f64(q), kd, vd, 32 ** -0.5, lambda j: 45)
        # each row's share of the error goes by its own size, not by the largest row's
        share, _ = attend(f64(q), kd, np.abs(vd).max(-1, keepdims=True) + 0 * vd, 32 ** -0.5, lambda j: 45)
        eps = torch.finfo(q.dtype).eps
        tol = (2.0 ** -18 if dtype == "f32" else eps / 2 + 3 * 2.0 ** -12) + 2 * score_error(f64(q), kd, 32 ** -0.5)
        np.testing.assert_allclose(f64(out), want, rtol=0, atol=tol * share.max())


@gpu
def test_scores_of_extreme_queries():
    # queries of 2^-100 and 2^100 keep their own scaling; a NaN query spoils its own row only
    rng = np.random.default_rng(4)
    cache = Cache(1, 3, 16, 1, 64)
    ks, vs = filled(rng, cache, [40])
    q = typed(rng, (1, 8, 64), "f32")
    q[0, 1] *= 2.0 ** -100
    q[0, 2] *= 2.0 ** 40
    q[0, 3] = 0.0
    q[0, 4, 5] = float("nan")
    out, lse, _ = attention(cache, q.cuda(), [0], [1], [40], 0.125, 0, "f32")
    want, wl = attend(f64(q), ks[0], vs[0], 0.125, lambda j: 40)
    for j in (0, 1, 2, 3, 5, 6, 7):   # row 2's weights are one-hot: its score errors do not reach the output
        dx = 0.0 if j == 2 else score_error(f64(q)[:, j:j + 1], ks[0], 0.125)
        np.testing.assert_allclose(f64(out)[0, j], want[0, j], atol=(2.0 ** -18 + 2 * dx) * np.abs(vs[0]).max())
    assert np.isnan(f64(out)[0, 4]).all() and np.isnan(f64(lse)[0, 4])


@gpu
def test_strided_queries_and_outputs():
    rng = np.random.default_rng(6)
    cache = Cache(3, 2, 16, 2, 64)
    filled(rng, cache, [20, 32, 9])
    q = typed(rng, (3, 4, 64), "f16").cuda()
    wide = torch.zeros(3, 3, 4, 64, dtype=torch.float16, device="cuda")
    wide[:, 0] = q
    out = torch.full((4, 3, 64), 7.0, dtype=torch.float16, device="cuda").transpose(0, 1)   # head-major storage
    a, la, _ = attention(cache, q, [0, 1, 2], [1] * 3, [20, 32, 9], 0.125, 0, "f16")
    b, lb, _ = attention(cache, wide[:, 0], [0, 1, 2], [1] * 3, [20, 32, 9], 0.125, 0, "f16", out=out)
    assert torch.equal(a, b) and torch.equal(la, lb)


@gpu
@pytest.mark.parametrize("q_len,kv_len,q_start", [(3, 20, 0), (1, 33, 0), (1, -1, 0), (-1, 20, 0), (1, 20, 2), (1, 20, -1)])
def test_bad_lengths_are_left_out_and_reported(q_len, kv_len, q_start):
    rng = np.random.default_rng(1)
    cache = Cache(2, 2, 16, 1, 64)
    filled(rng, cache, [20, 20])
    q = typed(rng, (2, 1, 64), "f32").cuda()
    good, _, _ = attention(cache, q, [0, 1], [0, 1], [20, 20], 0.125, 0, "f32", max_q=2, max_kv=32)
    assert status_bits() == 0
    out, lse, _ = attention(cache, q, [q_start, 1], [q_len, 1], [kv_len, 20], 0.125, 0, "f32", max_q=2, max_kv=32)
    assert status_bits() == 4
    assert torch.equal(out[1], good[1]) and bool((out[0] == 7).all()) and bool((lse[0] == 7).all())


@gpu
def test_pages_past_2_gib():
    # 2.4 GiB of pages, the sequence's in the last of them
    rng = np.random.default_rng(12)
    t, hk, d = 32, 8, 128
    per_page = 8 * 32 * 136
    n_pages = (5 << 29) // per_page
    cache = Cache(1, 2, t, hk, d, extra=0)
    cache.n_pages = n_pages
    cache.pages = torch.empty(n_pages * per_page, dtype=torch.uint8, device="cuda")
    cache.table = np.array([[n_pages - 1, n_pages - 2]], np.int32)
    cache.table_dev = torch.from_numpy(cache.table).cuda()
    check(cache, rng, [50], [1], hk, "bf16", 0)


@gpu
def test_two_streams_and_a_captured_step():
    # append + attention captured once and replayed on new rows gives what the
    # eager calls give, also while another stream works on another cache
    lib, rng = L.load(), np.random.default_rng(9)
    t, hk, d, n = 16, 2, 64, 40
    rows = [typed(rng, (1, hk, d), "bf16").cuda() for _ in range(6)]
    k, v, q = (torch.zeros(1, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    caches = [Cache(1, 4, t, hk, d, seed=2) for _ in range(3)]
    filled(rng, caches[0], [n])
    for c in caches[1:]:
        c.pages.copy_(caches[0].pages)

    def step(cache, at, stream):
        kv_len = ints([n + 1])
        out, lse = torch.empty_like(q), torch.empty(1, hk, device="cuda")
        rs = rows_struct(k, v, [0], [1], [at], 1, L.MC_BF16)
        a = L.Kv4AttentionArgs(q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), q_start=rs.keep[2].data_ptr(),
                               q_len=rs.keep[3].data_ptr(), kv_len=kv_len.data_ptr(), q_rows=1, q_row_stride=hk * d,
                               q_head_stride=d, out_row_stride=hk * d, out_head_stride=d, dtype=L.MC_BF16, heads=hk,
                               max_q_len=1, max_kv_len=64, causal=1, scale=0.125)
        cs = cache.struct()
        need = lib.mc_kv4_attention_workspace(C.byref(cs), C.byref(a))
        ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), need

        def go():
            assert lib.mc_kv4_append(C.byref(cs), C.byref(rs), stream.cuda_stream) == L.MC_OK
            assert lib.mc_kv4_attention(C.byref(cs), C.byref(a), stream.cuda_stream) == L.MC_OK
        return go, out, [rs, a, ws, lse, kv_len, cs]

    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    go0, out0, keep0 = step(caches[0], n, torch.cuda.current_stream())
    go1, out1, keep1 = step(caches[1], n, side)
    go2, out2, keep2 = step(caches[2], n, other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        go1()
    for i in range(3):
        k.copy_(rows[i]), v.copy_(rows[i + 1]), q.copy_(rows[i + 3])
        torch.cuda.synchronize()
        go0()
        graph.replay()
        go2()
        torch.cuda.synchronize()
        assert torch.equal(out0, out1) and torch.equal(out0, out2)
        assert torch.equal(caches[0].pages, caches[1].pages)
    assert status_bits() == 0


def test_key_counts_next_to_the_largest_integer():
    # a tile's last position has to be an int too
    lib, (cache, _, att) = L.load(), host_args()
    cache.page_tokens, cache.pages_per_seq = 8, 2**28 - 1
    att.max_kv_len = 2**31 - 256
    assert lib.mc_kv4_attention_workspace(C.byref(cache), C.byref(att)) > 0
    for n in (2**31 - 255, 2**31 - 8):
        att.max_kv_len = n
        assert lib.mc_kv4_attention_workspace(C.byref(cache), C.byref(att)) == 0
        assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_INVALID_INPUT


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -17, 2.0 ** -15, 2.0 ** -13, 2.0 ** -11])
def test_small_value_rows(dtype, size):
    # scales around f16's smallest normal number, 2^-14, and far into its subnormals: a row's largest
    # weight is taken with its scale and has to fit f16 all the same.  f16 outputs this small are
    # multiples of 2^-24: 2^-25 more.
    lib, rng = L.load(), np.random.default_rng(21)
    lens = [1, 45, 700]
    cache = Cache(3, 44, 16, 1, 64)
    k, v = typed(rng, (sum(lens), 1, 64), "f32"), typed(rng, (sum(lens), 1, 64), "f32", size)
    start = np.cumsum(lens) - lens
    cs = cache.struct()
    assert call(lib.mc_kv4_append, cs, rows_struct(k.cuda(), v.cuda(), start, lens, [0] * 3, 700, L.MC_F32)) == L.MC_OK
    kd, vd = ((lambda c, s, m: m.astype(float)[..., None] + s.astype(float)[..., None] * c)(*quantize(f64(x))) for x in (k, v))
    for q_size in (1.0, 20.0):
        q = typed(rng, (3, 2, 64), dtype, q_size)
        out, _, _ = attention(cache, q.cuda(), [0, 1, 2], [1] * 3, lens, 0.125, 0, dtype)
        eps = torch.finfo(q.dtype).eps
        for i, n in enumerate(lens):
            ki, vi = kd[start[i]:start[i] + n], vd[start[i]:start[i] + n]
            want, _ = attend(f64(q)[i:i + 1], ki, vi, 0.125, lambda j: n)
            tol = (2.0 ** -18 if dtype == "f32" else eps / 2 + 2.0 ** -11) + 2 * score_error(f64(q)[i:i + 1], ki, 0.125)
            np.testing.assert_allclose(f64(out)[i:i + 1], want, rtol=0,
                                       atol=tol * np.abs(vi).max() + (2.0 ** -25 if dtype == "f16" else 0.0))
    assert status_bits() == 0


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [110, 117, 118, 122, 126])
def test_queries_up_to_the_largest_number(dtype, exponent):
    # scores of 2^exponent are finite, and their weights one-hot: the output is one value row, to the
    # type's rounding (f32: 2^-20, as the row's parts of up to 3 max|v| are within 2^-22 each).
    # lse: 22-bit products (2^-21 of their sizes, of up to 3 max|k|).
    rng = np.random.default_rng(exponent)
    cache = Cache(1, 3, 16, 1, 64)
    ks, vs = filled(rng, cache, [40])
    q = torch.zeros(1, 2, 64)
    q[0, 0, :3] = torch.tensor([1.0, -0.5, 0.75]) * 2.0 ** exponent
    q[0, 1, 60:] = torch.tensor([-1.75, 0.0, 0.5, 1.5]) * 2.0 ** exponent
    q = q.to(DTYPES[dtype][0])
    out, lse, _ = attention(cache, q.cuda(), [0], [1], [40], 0.125, 0, dtype)
    want, wl = attend(f64(q), ks[0], vs[0], 0.125, lambda j: 40)
    tol = (2.0 ** -20 if dtype == "f32" else 2.0 ** -8 + 2.0 ** -11) * np.abs(vs[0]).max()
    np.testing.assert_allclose(f64(out), want, rtol=0, atol=tol)
    np.testing.assert_allclose(f64(lse), wl, rtol=0, atol=score_error(f64(q), ks[0], 0.125))


@gpu
@pytest.mark.parametrize("dtype,n,mean,spread,d,group", [
    ("f32", 65536, 1.0, 0.1, 64, 1), ("f32", 65536, -1.0, 0.1, 48, 3), ("f32", 262144, 0.0, 1.0, 64, 1),
    ("f32", 262144, 0.0, 1.0, 128, 8),
    ("f16", 262144, 0.0, 1.0, 64, 1), ("bf16", 262144, 0.0, 1.0, 64, 1), ("f16", 262144, 0.0, 1.0, 80, 16)])
def test_long_caches_of_many_sequences(dtype, n, mean, spread, d, group):
    # So many sequences that no keys are cut into ranges: one warp sums them all.  Sums in f32 round to
    # nearest, 2^-24.8 of the partial sum (root mean square) for each of n / 32 tiles, and for each of n / 8
    # weights of eight lanes: 2^-19.3 of the whole at 65,536 keys and 2^-18.3 at 262,144.  f32 outputs:
    # 2^-18 max|v| (root mean square), of values with a mean, whose sums grow with the keys.  16 bits, of
    # values without one: the output's rounding, 2^-18 max|v| for the sums (which are 2^-6 of that size)
    # and the weights' rounding, 2^-12.8 |v| / sqrt(n / 2.7) and so below 2^-20.
    lib, b = L.load(), 1200
    g = torch.Generator(device="cuda")
    g.manual_seed(d)
    one = Cache(1, n // 32, 32, 1, d, extra=0)
    k, v = (torch.randn(n, 1, d, generator=g, device="cuda") for _ in range(2))
    v = v * spread + mean
    cs = one.struct()
    assert call(lib.mc_kv4_append, cs, rows_struct(k, v, [0], [n], [0], n, L.MC_F32)) == L.MC_OK
    assert call(lib.mc_kv4_read, cs, rows_struct(k, v, [0], [n], [0], n, L.MC_F32)) == L.MC_OK
    one.b, one.table_dev = b, one.table_dev.expand(b, n // 32).contiguous()   # every sequence reads the same pages
    q = torch.randn(b, group, d, generator=g, device="cuda").to(DTYPES[dtype][0])
    out, lse, need = attention(one, q, np.arange(b), [1] * b, [n] * b, d ** -0.5, 0, dtype)
    assert need == 0 and status_bits() == 0
    at = [0, 1, b // 2, b - 1]
    x = q[at].double().reshape(-1, d) @ k[:, 0].double().T * d ** -0.5
    want = torch.softmax(x, 1) @ v[:, 0].double()
    got, big = out[at].double().reshape(-1, d), float(v.abs().max())
    if dtype == "f32":
        assert float((got - want).square().mean().sqrt()) <= 2.0 ** -18 * big
    else:
        assert bool(((got - want).abs() <= torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -18 * big).all())
    np.testing.assert_allclose(lse[at].double().reshape(-1).cpu(), torch.logsumexp(x, 1).cpu(), rtol=2.0 ** -18)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nats,at", [(17.4, 0), (17.4, 40000), (16.0, 9), (5.5, 200)])
def test_a_long_tail_behind_one_key(dtype, nats, at):
    # One key `nats` above 65,535 equal ones, whose weights count together; so many sequences that one warp
    # sums them all.  A lane adds up its four weights of a tile before they meet its sum: 2^11 roundings of
    # 2^-24 of the largest weight, which is nearly the whole sum, in one of eight lanes.  The key that stands
    # out has the value 0, so the output is as far off as the sum, and its type's rounding.
    lib, b, n, d = L.load(), 1200, 65536, 64
    rng = np.random.default_rng(at)
    one = Cache(1, n // 32, 32, 1, d, extra=0)
    k = torch.zeros(n, 1, d, device="cuda")
    k[at, 0, 0] = nats
    v = torch.from_numpy(rng.uniform(0.5, 1.5, (n, 1, d)).astype(np.float32)).cuda()
    v[at] = 0.0
    cs = one.struct()
    assert call(lib.mc_kv4_append, cs, rows_struct(k, v, [0], [n], [0], n, L.MC_F32)) == L.MC_OK
    assert call(lib.mc_kv4_read, cs, rows_struct(k, v, [0], [n], [0], n, L.MC_F32)) == L.MC_OK
    one.b, one.table_dev = b, one.table_dev.expand(b, n // 32).contiguous()
    q = torch.zeros(b, 1, d, dtype=DTYPES[dtype][0], device="cuda")
    q[:, 0, 0] = 8.0
    out, lse, need = attention(one, q, np.arange(b), [1] * b, [n] * b, 0.125, 0, dtype)
    assert need == 0 and status_bits() == 0
    x = k[:, 0, 0].double()
    want = torch.softmax(x, 0) @ v[:, 0].double()
    rounding = 2.0 ** -18 if dtype == "f32" else torch.finfo(q.dtype).eps / 2 + 2.0 ** -11
    assert bool(((out[:, 0].double() - want).abs() <= (2.0 ** -13 + rounding) * want).all())
    np.testing.assert_allclose(f64(lse), float(torch.logsumexp(x, 0)), rtol=2.0 ** -20, atol=2.0 ** -13)


def test_overlaps_of_wide_strides_are_refused():
    # (rows - 1) * row_stride or (heads - 1) * head_stride pass 64 bits, and what is left of them looks small
    lib = L.load()
    sound = L.MC_INVALID_INPUT if torch.cuda.is_available() else L.MC_CUDA   # past the checks; there is no such memory
    for rows, heads, row_stride, head_stride, want in (
            (2**30 + 1, 65536, 2**34, 2**19, L.MC_INVALID_INPUT),   # head 2^15 of a row is head 0 of the next
            (2**30 + 1, 65536, 2**34, 2**18, sound),                # 65,536 heads within the row's stride
            (2**30 + 1, 4, 2**34, 64, sound)):
        cache, r, att = host_args()
        cache.batch, cache.kv_heads = 1, heads
        att.heads, att.q_rows, att.out_row_stride, att.out_head_stride = heads, rows, row_stride, head_stride
        att.max_q_len = 1
        assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == want
        r.rows, r.k_row_stride, r.k_head_stride, r.v_row_stride, r.v_head_stride = rows, row_stride, head_stride, row_stride, head_stride
        assert lib.mc_kv4_read(C.byref(cache), C.byref(r), None) == want
    # more heads than a cache has: 2^31 - 2 of them, 2^33 apart
    cache, r, att = host_args()
    cache.batch, cache.kv_heads, att.max_q_len = 1, 1, 1
    att.heads, att.q_rows, att.out_row_stride, att.out_head_stride = 2**30 - 1, 2**20, 64, 2**34 + 64
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == sound
    att.out_row_stride = 2**20
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_INVALID_INPUT
    # strides whose bytes pass 64 bits
    for stride in (2**62, 2**61 + 64, 2**40):
        cache, r, att = host_args()
        att.q_row_stride = stride
        assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_INVALID_INPUT


def test_scales_past_the_largest_power_of_two_are_refused():
    # scores are taken in powers of two: scale * log2(e) has to be a number
    for scale, sound in ((2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False)):
        cache, _, att = host_args()
        att.scale = scale
        got = L.load().mc_kv4_attention(C.byref(cache), C.byref(att), None)
        assert got == (L.MC_CUDA if sound and not torch.cuda.is_available() else L.MC_INVALID_INPUT)


def test_tensors_of_no_rows_may_be_null():
    lib = L.load()
    sound = L.MC_INVALID_INPUT if torch.cuda.is_available() else L.MC_CUDA   # past the checks; there is no such memory
    cache, rows, att = host_args()
    rows.k, rows.v, rows.rows = None, None, 0
    att.q, att.out, att.q_rows = None, None, 0
    cache.pages, cache.n_pages = None, 0
    assert lib.mc_kv4_append(C.byref(cache), C.byref(rows), None) == sound
    assert lib.mc_kv4_read(C.byref(cache), C.byref(rows), None) == sound
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == sound
    rows.rows = att.q_rows = 1
    assert lib.mc_kv4_read(C.byref(cache), C.byref(rows), None) == L.MC_INVALID_INPUT
    assert lib.mc_kv4_attention(C.byref(cache), C.byref(att), None) == L.MC_INVALID_INPUT


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-30, 1.5])
def test_scales_of_any_sign(dtype, scale):
    rng = np.random.default_rng(31)
    cache = Cache(2, 9, 16, 2, 64)
    ks, vs = filled(rng, cache, [140, 77])
    q = typed(rng, (8, 4, 64), dtype)
    out, lse, _ = attention(cache, q.cuda(), [0, 4], [4, 4], [140, 77], scale, 1, dtype)
    for i, n in enumerate((140, 77)):
        at = slice(4 * i, 4 * i + 4)
        want, wl = attend(f64(q)[at], ks[i], vs[i], float(np.float32(scale)), lambda j: n - (3 - j))
        dx = score_error(f64(q)[at], ks[i], abs(scale))
        tol = (2.0 ** -18 if dtype == "f32" else torch.finfo(q.dtype).eps / 2 + 2.0 ** -11) + 2 * dx
        np.testing.assert_allclose(f64(out)[at], want, rtol=0, atol=tol * np.abs(vs[i]).max())
        np.testing.assert_allclose(f64(lse)[at], wl, rtol=2.0 ** -20, atol=2.0 ** -19 + dx)
