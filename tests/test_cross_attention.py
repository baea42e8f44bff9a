"""mc_cross_attention against a plain 64-bit form: packed and padded batches,
single tokens, shared heads and keys, masks, odd head sizes and lengths, split
keys, strides, infinities and NaN where the mask leaves keys out.

Tolerances, derived from the arithmetic.  f32: a product of three tf32 halves
is within 2^-21 of its value and a score's f32 sum loses at most 2^-21 more of
sum|q||k|: dx = 2^-20 * scale * sum|q| max|k|, which moves an output by at most
2 dx max|v|; the weighted sum and the sum of weights lose 2^-19 of max|v| each.
16 bits: products are exact; weights and output are rounded to the type, half
a step each: (eps / 2 + eps / 2 + 2 dx) max|v|.  The f32 errors are
independent, so their root mean square stays below 2^-19 max|v|.
"""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from marian_cuda import _lib as L  # noqa: E402

gpu = pytest.mark.gpu
DTYPES = {"f32": (torch.float32, L.MC_F32), "f16": (torch.float16, L.MC_F16), "bf16": (torch.bfloat16, L.MC_BF16)}


def attend(q, k, v, scale, live):
    """q [m, h, d], k, v [n, hk, d] float64, live [n] -> out [m, h, d], lse [m, h]."""
    m, h, d = q.shape
    k, v = k[live], v[live]
    out, lse = np.zeros((m, h, d)), np.full((m, h), -np.inf)
    if k.shape[0] == 0:
        return out, lse
    for j in range(h):
        x = q[:, j] @ k[:, j * k.shape[1] // h].T * scale
        top = x.max(1, keepdims=True)
        w = np.exp(x - top)
        out[:, j] = w @ v[:, j * k.shape[1] // h] / w.sum(1, keepdims=True)
        lse[:, j] = top[:, 0] + np.log(w.sum(1))
    return out, lse


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def typed(rng, shape, dtype, size=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * size).astype(np.float32)).to(DTYPES[dtype][0])


def f64(x):
    return x.float().cpu().numpy().astype(np.float64)


def status_bits():
    bits = C.c_uint32(0)
    assert L.load().mc_op_status(C.byref(bits)) == L.MC_OK
    return bits.value


def arguments(q, k, v, out, lse, lens, mask, dtype, scale, max_q, max_k):
    a = L.CrossAttentionArgs(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), lse=None if lse is None else lse.data_ptr(),
        q_start=lens[0].data_ptr(), q_len=lens[1].data_ptr(), k_start=lens[2].data_ptr(), k_len=lens[3].data_ptr(),
        key_mask=None if mask is None else mask.data_ptr(), q_rows=q.shape[0], k_rows=k.shape[0],
        q_row_stride=q.stride(0), q_head_stride=q.stride(1), k_row_stride=k.stride(0), k_head_stride=k.stride(1),
        v_row_stride=v.stride(0), v_head_stride=v.stride(1), out_row_stride=out.stride(0),
        out_head_stride=out.stride(1), dtype=DTYPES[dtype][1], batch=lens[0].shape[0], heads=q.shape[1],
        kv_heads=k.shape[1], head_dim=q.shape[2], max_q_len=max_q, max_k_len=max_k, scale=scale)
    need = L.load().mc_cross_attention_workspace(C.byref(a))
    ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    a.keep = (ws, lens, mask, q, k, v, out, lse)
    return a, need


def run(q, k, v, q_start, q_len, k_start, k_len, dtype, scale, mask=None, max_q=None, max_k=None, out=None):
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    lens = [ints(x) for x in (q_start, q_len, k_start, k_len)]
    m = None if mask is None else torch.from_numpy(np.asarray(mask, np.uint8)).cuda()
    a, need = arguments(q, k, v, out, lse, lens, m, dtype, scale, int(max(q_len)) if max_q is None else max_q,
                        int(max(k_len)) if max_k is None else max_k)
    torch.cuda.synchronize()
    assert L.load().mc_cross_attention(C.byref(a), torch.cuda.current_stream().cuda_stream) == L.MC_OK
    torch.cuda.synchronize()
    return out, lse, need


def compare(q, k, v, out, lse, q_start, q_len, k_start, k_len, dtype, scale, mask=None):
    qd, kd, vd, od, ld = (f64(x) for x in (q, k, v, out, lse))
    eps = torch.finfo(q.dtype).eps
    touched = np.zeros(q.shape[0], bool)
    for q0, m, k0, n in zip(q_start, q_len, k_start, k_len):
        at = slice(q0, q0 + m)
        touched[at] = True
        if m == 0:
            continue
        live = np.ones(n, bool) if mask is None else np.asarray(mask[k0:k0 + n]) != 0
        want, wl = attend(qd[at], kd[k0:k0 + n], vd[k0:k0 + n], scale, live)
        some = live.any()
        big = np.abs(vd[k0:k0 + n][live]).max() if some else 1.0
        dx = 2.0 ** -20 * scale * np.abs(qd[at]).sum(-1).max() * np.abs(kd[k0:k0 + n][live]).max() if some else 0.0
        tol = (2.0 ** -18 if dtype == "f32" else eps) + 2 * dx
        np.testing.assert_allclose(od[at], want, rtol=0, atol=tol * big)
        if dtype == "f32":
            assert np.sqrt(np.mean((od[at] - want) ** 2)) <= 2.0 ** -19 * big
        np.testing.assert_allclose(ld[at], wl, rtol=2.0 ** -20, atol=2.0 ** -19 + dx)
    assert (od[~touched] == 7).all() and (ld[~touched] == 7).all()


def check(rng, q_len, k_len, h, hk, d, dtype, mask=None, gap_q=0, gap_k=0, size=1.0):
    b = len(q_len)
    q_start = np.cumsum(q_len) - q_len + gap_q * np.arange(b)
    k_start = np.cumsum(k_len) - k_len + gap_k * np.arange(b)
    rows_q, rows_k = int(np.sum(q_len)) + gap_q * b + 1, int(np.sum(k_len)) + gap_k * b + 1
    q, k, v = typed(rng, (rows_q, h, d), dtype, size), typed(rng, (rows_k, hk, d), dtype), typed(rng, (rows_k, hk, d), dtype)
    m = None
    if mask is not None:
        m = (rng.random(rows_k) < mask).astype(np.uint8)
        m[k_start[0]:k_start[0] + k_len[0]] = 0     # nothing left of the first
    # what no query may see is not finite
    seen = np.zeros(rows_k, bool)
    for k0, n in zip(k_start, k_len):
        seen[k0:k0 + n] = True if m is None else m[k0:k0 + n] != 0
    lost = torch.from_numpy(~seen)
    k[lost], v[lost] = float("nan"), float("inf")
    scale = d ** -0.5
    out, lse, need = run(q.cuda(), k.cuda(), v.cuda(), q_start, q_len, k_start, k_len, dtype, scale, m)
    assert status_bits() == 0
    compare(q, k, v, out, lse, q_start, q_len, k_start, k_len, dtype, scale, m)
    return need


# ---- refusals ------------------------------------------------------------------

def host_args():
    return L.CrossAttentionArgs(q=1 << 20, k=2 << 20, v=3 << 20, out=4 << 20, lse=64, q_start=64, q_len=64, k_start=64,
                                k_len=64, workspace=1 << 20, workspace_bytes=1 << 40, q_rows=10, k_rows=20,
                                q_row_stride=256, q_head_stride=64, k_row_stride=128, k_head_stride=64,
                                v_row_stride=128, v_head_stride=64, out_row_stride=256, out_head_stride=64,
                                dtype=L.MC_F32, batch=2, heads=4, kv_heads=2, head_dim=64, max_q_len=5, max_k_len=10,
                                scale=0.125)


@pytest.mark.parametrize("field,value", [
    ("q", 0), ("k", 0), ("v", 0), ("out", 0), ("q", (1 << 20) + 8), ("k", (2 << 20) + 4), ("out", 1 << 20),
    ("out", 2 << 20), ("out", 3 << 20), ("lse", 2), ("q_start", 0), ("q_len", 0), ("k_start", 0), ("k_len", 0),
    ("k_len", 66), ("q_rows", -1), ("k_rows", -1), ("k_rows", 1 << 31), ("q_row_stride", 254), ("k_row_stride", -128),
    ("v_head_stride", 62), ("out_head_stride", 32), ("out_row_stride", 64), ("out_row_stride", 0), ("dtype", 3),
    ("dtype", -1), ("batch", -1), ("heads", 3), ("heads", 0), ("kv_heads", 0), ("kv_heads", -2), ("head_dim", 24),
    ("head_dim", 0), ("head_dim", 144), ("max_q_len", -1), ("max_k_len", -1), ("scale", float("nan")),
    ("scale", float("-inf"))])
def test_bad_arguments_are_refused(field, value):
    a = host_args()
    setattr(a, field, value)
    assert L.load().mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT


def test_strides_of_16_bit_rows_are_checked_in_bytes():
    a = host_args()
    a.dtype, a.k_row_stride = L.MC_BF16, 132   # 264 bytes
    assert L.load().mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT


def test_null_empty_and_short_workspace():
    lib = L.load()
    assert lib.mc_cross_attention(None, None) == L.MC_INVALID_INPUT
    assert lib.mc_cross_attention_workspace(None) == 0
    for field in ("batch", "max_q_len"):
        a = host_args()
        setattr(a, field, 0)
        assert lib.mc_cross_attention(C.byref(a), None) == L.MC_OK
    a = host_args()
    a.batch, a.max_q_len, a.max_k_len = 1, 1, 20000
    need = lib.mc_cross_attention_workspace(C.byref(a))
    assert need > 0
    for ws, n in ((0, need), (1 << 20, need - 1), ((1 << 20) + 4, need)):
        a.workspace, a.workspace_bytes = ws, n
        assert lib.mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT
    if not torch.cuda.is_available():
        assert lib.mc_cross_attention(C.byref(host_args()), None) == L.MC_CUDA


@gpu
def test_host_memory_is_refused():
    a = host_args()
    host = torch.zeros(4096)
    a.q = (host.data_ptr() + 15) // 16 * 16
    assert L.load().mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT


# ---- the definition --------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128])
def test_single_tokens(dtype, d):
    rng = np.random.default_rng(d)
    k_len = [1, 0, 7, 31, 32, 33, 63, 64, 65, 127, 256]
    check(rng, [1] * len(k_len), k_len, 2, 2, d, dtype, gap_k=1)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,hk,group", [(64, 2, 1), (48, 1, 8), (128, 2, 4), (80, 3, 7), (16, 1, 3)])
@pytest.mark.parametrize("top", [3, 30, 200])
def test_ragged_batches_with_shared_heads(dtype, d, hk, group, top):
    rng = np.random.default_rng(d + top)
    q_len = [top, 1, 0, 2, max(1, top // 2 + 1)]
    k_len = [3, 200, 40, 0, 65]
    check(rng, q_len, k_len, hk * group, hk, d, dtype, gap_q=2, gap_k=3)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,q_len", [(64, 1), (48, 20), (128, 70), (96, 33)])
def test_padded_batches_with_masks(dtype, d, q_len):
    rng = np.random.default_rng(q_len)
    check(rng, [q_len, q_len, q_len, q_len - 1], [100, 130, 64, 1], 4, 2, d, dtype, mask=0.6, gap_q=4, gap_k=30)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_len,k_len,h,hk", [([1], [1000], 1, 1), ([1, 1], [2500, 3], 8, 2), ([5], [4097], 2, 2),
                                             ([40, 40], [3000, 0], 2, 1), ([1], [300], 8, 8)])
def test_split_keys(dtype, q_len, k_len, h, hk):
    rng = np.random.default_rng(k_len[0])
    for mask in (None, 0.5):
        if mask is None or len(q_len) > 1:
            check(rng, q_len, k_len, h, hk, 64, dtype, mask=mask)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,q_len,k_len,h,hk", [(128, [300, 129], [1000, 257], 4, 2), (64, [513], [640], 2, 2),
                                               (48, [128, 128], [129, 4095], 2, 1), (112, [255], [128], 2, 2),
                                               (96, [700], [1], 1, 1), (16, [256], [333], 2, 2), (32, [600], [513], 4, 4),
                                               (80, [1000, 5, 400], [700, 900, 0], 2, 2)])
def test_long_sequences(dtype, d, q_len, k_len, h, hk):
    rng = np.random.default_rng(d)
    check(rng, q_len, k_len, h, hk, d, dtype, gap_q=1, gap_k=2)
    check(rng, q_len, k_len, h, hk, d, dtype, gap_q=1, gap_k=2, size=6.0)   # weights near one-hot


@gpu
def test_long_sequences_with_masks():
    rng = np.random.default_rng(3)
    check(rng, [300, 300], [400, 700], 2, 2, 64, "bf16", mask=0.5)


@gpu
def test_split_keys_take_a_workspace_and_small_calls_none():
    rng = np.random.default_rng(2)
    assert check(rng, [1], [4000], 1, 1, 64, "bf16") > 0
    assert check(rng, [1] * 64, [64] * 64, 8, 8, 64, "bf16") == 0


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_several_queries_share_one_source(dtype):
    rng = np.random.default_rng(1)
    q, k, v = typed(rng, (12, 4, 64), dtype), typed(rng, (50, 4, 64), dtype), typed(rng, (50, 4, 64), dtype)
    q_start, q_len, k_start, k_len = [0, 5, 6], [5, 1, 6], [3, 3, 10], [40, 40, 33]
    out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), q_start, q_len, k_start, k_len, dtype, 0.125)
    compare(q, k, v, out, lse, q_start, q_len, k_start, k_len, dtype, 0.125)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_len", [1, 20, 300])
def test_strides_and_head_major_layouts(dtype, q_len):
    rng = np.random.default_rng(q_len)
    h, d, n = 4, 64, 150
    q = typed(rng, (h, q_len, d), dtype).cuda().transpose(0, 1)          # head-major
    kv = typed(rng, (n, 2, h, d), dtype).cuda()                          # interleaved
    wide = torch.full((q_len, h, d + 16), 7.0, dtype=q.dtype, device="cuda")
    args = ([0], [q_len], [0], [n], dtype, 0.125)
    a, la, _ = run(q.contiguous(), kv[:, 0].contiguous(), kv[:, 1].contiguous(), *args)
    b, lb, _ = run(q, kv[:, 0], kv[:, 1], *args, out=wide[:, :, :d])
    assert torch.equal(a, b) and torch.equal(la, lb) and bool((wide[:, :, d:] == 7).all())
    # one key/value row for every head (stride 0)
    one = kv[:, 0, :1].expand(n, h, d)
    c, _, _ = run(q, one, one, *args)
    e, _, _ = run(q.contiguous(), one.contiguous(), one.contiguous(), *args)
    assert torch.equal(c, e)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_nan_query_spoils_its_own_row_only(dtype):
    rng = np.random.default_rng(7)
    for q_len in (4, 40, 200):
        q, k, v = typed(rng, (q_len, 2, 64), dtype), typed(rng, (90, 2, 64), dtype), typed(rng, (90, 2, 64), dtype)
        args = ([0], [q_len], [0], [90], dtype, 0.125)
        good, gl, _ = run(q.cuda(), k.cuda(), v.cuda(), *args)
        q[2, 1, 3] = float("nan")
        out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), *args)
        same = torch.ones(q_len, 2, dtype=torch.bool, device="cuda")
        same[2, 1] = False
        assert torch.equal(out[same], good[same]) and torch.equal(lse[same], gl[same])
        assert bool(out[2, 1].isnan().all()) and bool(lse[2, 1].isnan())


@gpu
@pytest.mark.parametrize("q_len", [1, 200])
def test_scores_far_from_zero(q_len):
    # every score near +-4000 (f32 keeps 2^-12 of those): the maximum has to follow
    rng = np.random.default_rng(9)
    for sign in (1.0, -1.0):
        q = torch.full((q_len, 1, 64), 2.0).to(torch.bfloat16)
        k = (torch.full((100, 1, 64), 250.0 * sign)).to(torch.bfloat16)
        v = typed(rng, (100, 1, 64), "bf16")
        out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), [0], [q_len], [0], [100], "bf16", 0.125)
        want = f64(v).mean(0)
        np.testing.assert_allclose(f64(out), np.broadcast_to(want, out.shape), atol=2.0 ** -8 * np.abs(f64(v)).max())
        np.testing.assert_allclose(f64(lse), 4000.0 * sign + np.log(100.0), rtol=2.0 ** -20)


@gpu
@pytest.mark.parametrize("field,value", [("q_start", -1), ("q_start", 9), ("q_len", -1), ("q_len", 4), ("k_start", -1),
                                         ("k_start", 12), ("k_len", 21), ("k_len", -5), ("k_start", 2147483647)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bad_lengths_are_left_out_and_reported(dtype, field, value):
    rng = np.random.default_rng(4)
    q, k, v = (typed(rng, (n, 2, 64), dtype).cuda() for n in (10, 30, 30))
    given = {"q_start": [0, 5], "q_len": [3, 3], "k_start": [0, 10], "k_len": [20, 20]}
    good, gl, _ = run(q, k, v, *given.values(), dtype, 0.125, max_q=3, max_k=20)
    assert status_bits() == 0
    given[field] = [value, given[field][1]]
    out, lse, _ = run(q, k, v, *given.values(), dtype, 0.125, max_q=3, max_k=20)
    assert status_bits() == 4
    assert torch.equal(out[5:8], good[5:8]) and torch.equal(lse[5:8], gl[5:8])
    rest = [i for i in range(10) if not 5 <= i < 8]
    assert bool((out[rest] == 7).all()) and bool((lse[rest] == 7).all())


@gpu
@pytest.mark.parametrize("dtype,q_len,k_len", [("f32", 1, 900), ("bf16", 1, 2000), ("bf16", 300, 500), ("f16", 20, 90)])
def test_captured_and_replayed_on_new_rows(dtype, q_len, k_len):
    lib, rng = L.load(), np.random.default_rng(11)
    q, k, v = (torch.zeros(n, 2, 64, dtype=DTYPES[dtype][0], device="cuda") for n in (q_len, k_len, k_len))
    out, lse = torch.zeros_like(q), torch.zeros(q_len, 2, device="cuda")
    a, _ = arguments(q, k, v, out, lse, [ints([0]), ints([q_len]), ints([0]), ints([k_len])], None, dtype, 0.125, q_len, k_len)
    run(q, k, v, [0], [q_len], [0], [k_len], dtype, 0.125)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        assert lib.mc_cross_attention(C.byref(a), side.cuda_stream) == L.MC_OK
    for _ in range(3):
        for x in (q, k, v):
            x.copy_(typed(rng, tuple(x.shape), dtype))
        graph.replay()
        torch.cuda.synchronize()
        want, wl, _ = run(q, k, v, [0], [q_len], [0], [k_len], dtype, 0.125)
        assert torch.equal(out, want) and torch.equal(lse, wl)
    # lse may be left out
    a.lse = None
    assert lib.mc_cross_attention(C.byref(a), None) == L.MC_OK


@gpu
def test_rows_past_2_gib():
    # keys whose byte offsets pass 2^32, the sequence's the last of them
    rng = np.random.default_rng(5)
    rows, hk, d = 300_000, 64, 128     # 16 KiB a row: 4.6 GiB
    k = torch.empty(rows, hk, d, dtype=torch.bfloat16, device="cuda")
    n = 70
    for q_len in (1, 140):
        q = typed(rng, (q_len, hk, d), "bf16")
        kv = typed(rng, (n, hk, d), "bf16")
        k[rows - n:] = kv.cuda()
        out, lse, _ = run(q.cuda(), k, k, [0], [q_len], [rows - n], [n], "bf16", d ** -0.5)
        compare(q, kv, kv, out, lse, [0], [q_len], [0], [n], "bf16", d ** -0.5)


@gpu
@pytest.mark.parametrize("h,hk,cut", [(16, 8, False), (6, 3, True)])
def test_long_sequences_in_several_waves(h, hk, cut):
    # units of 256 rows, 13 sequences of up to 1,024 rows a head: 416 (the last wave more than half
    # full) or 156, of which the keys of the last 8 are cut into ranges; among them a sequence without
    # keys, one with few, one with no queries
    rng = np.random.default_rng(6)
    need = check(rng, [512] * 9 + [300, 0, 257, 256], [1100] * 8 + [0, 900, 1100, 130, 1100], h, hk, 32, "bf16")
    assert (need > 0) == cut
    need = check(rng, [512] * 9 + [300, 0, 256, 257], [1100] * 11 + [130, 0], h, hk, 32, "bf16")
    assert (need > 0) == cut


def test_key_counts_next_to_the_largest_integer():
    # a tile's last position has to be an int too
    lib, a = L.load(), host_args()
    a.k_rows = a.max_k_len = 2**31 - 256
    assert lib.mc_cross_attention_workspace(C.byref(a)) > 0
    for n in (2**31 - 255, 2**31 - 1):
        a.k_rows = a.max_k_len = n
        assert lib.mc_cross_attention_workspace(C.byref(a)) == 0
        assert lib.mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT


@gpu
@pytest.mark.parametrize("d,q_len,n", [(64, 1, 90), (48, 20, 90), (128, 70, 90), (64, 1, 3000), (16, 2, 33)])
@pytest.mark.parametrize("case", ["k lowest", "k -inf", "v inf", "v -inf", "v largest", "v all large", "q largest", "k inf"])
@pytest.mark.parametrize("masked", [False, True])
def test_f32_infinities_and_largest_numbers(d, q_len, n, case, masked):
    # 64-bit arithmetic says what comes of them: a score of -inf (or far below the others) is a weight of 0,
    # an infinite value an infinite output, and a NaN only what has none.  Tolerances as in compare(), per
    # channel, since one channel may hold numbers of another size.
    rng = np.random.default_rng(d + n)
    q, k, v = (typed(rng, (m, 2, d), "f32") for m in (q_len, n, n))
    q = q.abs() + 0.1
    mask = None
    if masked:
        mask = (rng.random(n) < 0.7).astype(np.uint8)
        mask[5], mask[7] = 1, 0
        k[7], v[7] = float("inf"), float("nan")     # left out
    big = 3.4028234663852886e38
    if case == "k lowest":
        k[5, 0] = -big
    elif case == "k -inf":
        k[5, 0, 3] = -float("inf")
    elif case == "k inf":
        k[5, 0, 3] = float("inf")
    elif case == "v inf":
        v[5, 0, 3] = float("inf")
    elif case == "v -inf":
        v[5, 0, 2], v[5, 0, 3], v[2, 0, 3] = -float("inf"), -float("inf"), float("inf")
        if masked:
            mask[2] = 1
    elif case == "v largest":
        v[5, 0, 3], v[5, 0, 4] = big, -big
    elif case == "v all large":                     # sums of at most 3,000 weights of 1 stay in range
        v[:, 0, 3] = torch.from_numpy(rng.uniform(-1e34, 1e34, n).astype(np.float32))
    else:
        q[0, 0, 3] = big
        k[:, 0, 3] = torch.from_numpy(rng.uniform(-1e-38, 1e-38, n).astype(np.float32))
    scale = d ** -0.5
    out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), [0], [q_len], [0], [n], "f32", scale, mask)
    live = np.ones(n, bool) if mask is None else mask != 0
    with np.errstate(invalid="ignore", over="ignore"):
        want, wl = attend(f64(q), f64(k), f64(v), scale, live)
    got, finite_v = f64(out), np.where(np.isfinite(f64(v)), f64(v), 0.0)[live]
    small_k = np.where(np.abs(f64(k)) < 1e30, f64(k), 0.0)[live]
    small_q = np.where(np.abs(f64(q)) < 1e30, f64(q), 3.4)      # its products with k are at most that
    dx = 2.0 ** -20 * scale * np.abs(small_q).sum(-1).max() * max(1.0, np.abs(small_k).max())
    if case == "k inf":
        assert np.isnan(got[:, 0]).all() and np.isnan(f64(lse)[:, 0]).all()
        got, want, wl, lse = got[:, 1:], want[:, 1:], wl[:, 1:], lse[:, 1:]
        finite_v = finite_v[:, 1:]
    assert (np.isnan(got) == np.isnan(want)).all() and (np.isinf(got) == np.isinf(want)).all()
    for j in range(got.shape[1]):
        for c in range(d):
            w, g = want[:, j, c], got[:, j, c]
            some = np.isfinite(w)
            assert (g[np.isinf(w)] == w[np.isinf(w)]).all()
            np.testing.assert_allclose(g[some], w[some], rtol=0, atol=(2.0 ** -18 + 2 * dx) * np.abs(finite_v[:, j, c]).max())
    np.testing.assert_allclose(f64(lse), wl, rtol=2.0 ** -20, atol=2.0 ** -19 + dx)
    assert status_bits() == 0


def long_tail(dtype, b, nats, at, masked):
    """One key `nats` above 65,535 equal ones: each of those has a weight of some 2^-25 of the largest, all
    of them together count.  With 148 sequences no keys are cut into ranges.  16-bit weights are rounded to
    the type, and in f16 to 2^-24 at 2^7 (long tiles) or more times their size: 2^-32 of the largest.  Tiles of
    64 keys or more are added up in f32: at most 2^10 roundings of 2^-24 of the sum each, of which the key
    that stands out, whose value is 0, has no part in the output's numerator."""
    rng, n, m = np.random.default_rng(at), 65536, 128
    q, k = torch.zeros(m * b, 1, 64), torch.zeros(n, 1, 64)
    q[:, 0, 0], k[at, 0, 0] = 8.0, nats
    v = torch.from_numpy(rng.uniform(0.5, 1.5, (n, 1, 64)).astype(np.float32))
    v[at] = 0.0
    q, k, v = (x.to(DTYPES[dtype][0]) for x in (q, k, v))
    out, lse, need = run(q.cuda(), k.cuda(), v.cuda(), np.arange(b) * m, [m] * b, [0] * b, [n] * b, dtype, 0.125,
                         np.ones(n, np.uint8) if masked else None)
    w = np.exp(f64(k)[:, 0, 0] - f64(k)[at, 0, 0])
    want = w @ f64(v)[:, 0] / w.sum()
    tol = (torch.finfo(q.dtype).eps + 2.0 ** -13) * want + (n * 2.0 ** -32 * 1.5 if dtype == "f16" else 0.0)
    got = out.double().reshape(m * b, 64).cpu().numpy()
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    np.testing.assert_allclose(f64(lse), f64(k)[at, 0, 0] + np.log(w.sum()), rtol=2.0 ** -20, atol=2.0 ** -14)
    assert status_bits() == 0


LONG_TAILS = [(148, 17.4, 0), (148, 17.4, 40000), (148, 17.4, 65535), (148, 19.0, 100), (148, 5.5, 200),
              (148, 5.5, 65000), (1, 17.4, 30000)]


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("b,nats,at", LONG_TAILS)
def test_a_long_tail_behind_one_key(dtype, b, nats, at):
    long_tail(dtype, b, nats, at, False)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("b,nats,at", LONG_TAILS)
def test_a_long_tail_behind_one_key_with_a_mask(dtype, b, nats, at):
    long_tail(dtype, b, nats, at, True)


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,b,m,n,d", [
    ("f16", 460, 1, 262144, 64), ("f16", 460, 20, 262144, 48), ("f16", 148, 128, 262144, 64),
    ("f16", 150, 130, 100001, 128), ("bf16", 460, 1, 1048576, 64), ("bf16", 148, 128, 1048576, 64)])
def test_many_keys_of_one_sign(dtype, b, m, n, d, masked):
    # Equal weights, which are exact, over so many sequences that they fill the GPU: what is left is half a
    # step of the output, 2^-11 (f16) or 2^-8 for 1 to 2, and what the tensor cores' additions cut off, 2^-23
    # for each 16 keys of a range: 2^-13 of the output in 2^14 keys (f16), 2^-10 in 2^17 (bf16).
    g = torch.Generator(device="cuda")
    g.manual_seed(d)
    q = torch.zeros(b * m, 1, d, dtype=DTYPES[dtype][0], device="cuda")
    k = torch.randn(n, 1, d, generator=g, device="cuda").to(q.dtype)
    v = (torch.rand(n, 1, d, generator=g, device="cuda") * 0.8 + 1.0).to(q.dtype)
    k_len = np.full(b, n)
    k_len[1], k_len[3] = 40, 0          # sequences of one range and of none
    out, lse, need = run(q, k, v, np.arange(b) * m, [m] * b, [0] * b, k_len, dtype, d ** -0.5,
                         np.ones(n, np.uint8) if masked else None)
    assert need > 0 and status_bits() == 0
    want = torch.stack([v[:x, 0].double().mean(0) if x else torch.zeros(d, device="cuda", dtype=torch.float64) for x in k_len[:4]])
    want = want[torch.arange(b, device="cuda").clamp(max=4) % 4].repeat_interleave(m, 0)
    error = (out.double()[:, 0] - want).abs()
    share = 2.0 ** -13 if dtype == "f16" else 2.0 ** -10
    assert bool((error <= (2.0 ** -11 if dtype == "f16" else 2.0 ** -8) + share * want).all()), float(error.max())
    np.testing.assert_allclose(f64(lse)[:m], np.log(n), rtol=0, atol=2.0 ** -17)
    np.testing.assert_allclose(f64(lse)[-m:], np.log(n), rtol=0, atol=2.0 ** -17)
    assert np.isneginf(f64(lse)[3 * m:4 * m]).all()


def test_ranges_of_16_bit_keys_are_bounded():
    # the workspace follows the number of ranges: 512 units of 64 rows (small tiles) fill the GPU
    lib, a = L.load(), host_args()
    a.batch, a.heads, a.kv_heads, a.max_q_len, a.key_mask = 64, 8, 8, 64, 64
    slots = 64 * 8 * 64
    for dtype, most in ((L.MC_F32, None), (L.MC_F16, 1 << 14), (L.MC_BF16, 1 << 17)):
        a.dtype = dtype
        for n in (1, 1 << 14, (1 << 14) + 1, 1 << 17, (1 << 17) + 1, 1 << 20):
            a.max_k_len = a.k_rows = n
            ranges = 1 if most is None else -(-n // most)
            least = 0 if ranges == 1 else slots * ranges * (64 + 1) * 4
            got = lib.mc_cross_attention_workspace(C.byref(a))
            assert got >= least and (dtype != L.MC_F32 or got == 0)


def test_products_of_sizes_past_64_bits_are_refused():
    # 2^30 sequences x 2^16 heads x row tiles of 16 rows: (2^28 / 16 + 1) * 2^46 is past 2^63, and what a
    # 64-bit product keeps of it looks small
    lib = L.load()
    for batch, heads, max_q_len in ((2**30, 65536, 2**22 - 16), (2**30, 65536, 2**30 - 16), (2**16, 2**16, 1), (2**31 - 1, 2, 1)):
        a = host_args()
        a.batch, a.heads, a.kv_heads, a.max_q_len, a.q_rows = batch, heads, heads, max_q_len, 1
        assert lib.mc_cross_attention_workspace(C.byref(a)) == 0
        assert lib.mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT


def test_overlaps_of_wide_strides_are_refused():
    # (rows - 1) * row_stride passes 64 bits, and what is left of it looks small: head 2^15 of a row would be
    # head 0 of the next
    a = host_args()
    a.batch, a.heads, a.kv_heads, a.max_q_len, a.q_rows = 1, 65536, 65536, 1, 2**30 + 1
    a.out_row_stride, a.out_head_stride = 2**34, 2**19
    assert L.load().mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT
    a.out_head_stride = 2**18
    sound = L.MC_INVALID_INPUT if torch.cuda.is_available() else L.MC_CUDA   # past the checks; there is no such memory
    assert L.load().mc_cross_attention(C.byref(a), None) == sound


# ---- the long tiles' edges: 128 rows or more, two key tiles or more, 16 bits, no mask ----

@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("b,q_len,n,d", [(1, 128, 200, 64), (2, 300, 700, 128), (200, 130, 300, 64), (1, 260, 5000, 48)])
def test_long_tiles_keep_a_nan_query_to_its_row(dtype, b, q_len, n, d):
    rng = np.random.default_rng(n)
    q, k, v = typed(rng, (b * q_len, 2, d), dtype, 4.0), typed(rng, (n, 2, d), dtype), typed(rng, (n, 2, d), dtype)
    k *= torch.linspace(0.2, 2.0, n).to(k.dtype)[:, None, None]        # maxima grow on the way: rows are rescaled
    args = (np.arange(b) * q_len, [q_len] * b, [0] * b, [n] * b, dtype, d ** -0.5)
    good, gl, _ = run(q.cuda(), k.cuda(), v.cuda(), *args)
    spoilt = [(2, 1), (q_len - 1, 0), ((b - 1) * q_len + 65, 1), (b * q_len - 1, 0)]
    same = torch.ones(b * q_len, 2, dtype=torch.bool, device="cuda")
    for i, (row, head) in enumerate(spoilt):
        q[row, head, i * 7 % d] = float("nan")
        same[row, head] = False
    out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), *args)
    assert torch.equal(out[same], good[same]) and torch.equal(lse[same], gl[same])
    assert bool(out[~same].isnan().all()) and bool(lse[~same].isnan().all()) and bool(good.isfinite().all())


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_tiles_on_infinities(dtype):
    # a key whose score is -inf for every query weighs nothing; an infinite value makes its channel infinite
    rng, n, q_len = np.random.default_rng(3), 300, 150
    q, k, v = (typed(rng, (m, 2, 64), dtype) for m in (q_len, n, n))
    q = q.abs() + 0.1
    k[140, 0, 3], v[200, 1, 5], v[7, 1, 6] = -float("inf"), float("inf"), -float("inf")
    out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), [0], [q_len], [0], [n], dtype, 0.125)
    rest = np.ones(n, bool)
    rest[140] = False
    qd, kd, vd, od = (f64(x) for x in (q, k, v, out))
    want, wl = attend(qd, np.where(np.isfinite(kd), kd, 0.0), np.where(np.isfinite(vd), vd, 0.0), 0.125, rest)
    dx = 2.0 ** -20 * 0.125 * np.abs(qd).sum(-1).max() * np.abs(kd[np.isfinite(kd)]).max()
    tol = (torch.finfo(q.dtype).eps + 2 * dx) * np.abs(vd[np.isfinite(vd)]).max()
    np.testing.assert_allclose(od[:, 0], want[:, 0], rtol=0, atol=tol)
    np.testing.assert_allclose(f64(lse)[:, 0], wl[:, 0], rtol=2.0 ** -20, atol=2.0 ** -19 + dx)
    assert (od[:, 1, 5] == np.inf).all() and (od[:, 1, 6] == -np.inf).all() and np.isfinite(od[:, 1, 7:]).all()


@gpu
@pytest.mark.parametrize("dtype,size", [("bf16", 250.0), ("f16", 250.0), ("bf16", 250000.0)])
def test_long_tiles_on_scores_far_from_zero(dtype, size):
    # every score of a half near +-size * 16: equal scores share the weight, and the half below has none
    rng, n = np.random.default_rng(9), 300
    for high in (slice(0, 150), slice(150, 300), slice(100, 103)):
        q = torch.full((140, 1, 64), 2.0).to(DTYPES[dtype][0])
        k = torch.full((n, 1, 64), -size)
        k[high] = size
        k, v = k.to(q.dtype), typed(rng, (n, 1, 64), dtype)
        out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), [0], [140], [0], [n], dtype, 0.125)
        want, one = f64(v)[high].mean(0), f64(k)[high][0, 0, 0]
        np.testing.assert_allclose(f64(out), np.broadcast_to(want, out.shape),
                                   atol=torch.finfo(q.dtype).eps * np.abs(f64(v)).max())
        np.testing.assert_allclose(f64(lse), 16.0 * one + np.log(high.stop - high.start), rtol=2.0 ** -20)
        q[:] = -2.0     # now the other half is above
        out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), [0], [140], [0], [n], dtype, 0.125)
        rest = np.ones(n, bool)
        rest[high] = False
        np.testing.assert_allclose(f64(out), np.broadcast_to(f64(v)[rest].mean(0), out.shape),
                                   atol=torch.finfo(q.dtype).eps * np.abs(f64(v)).max())


@gpu
def test_long_tiles_past_4_gib():
    # keys and values whose byte offsets pass 2^32, the sequence's the last rows; several key tiles and a
    # rest, and heads at 2^31 bytes too
    rng, rows, hk, d, n = np.random.default_rng(5), 300_000, 64, 128, 333
    k = torch.empty(rows, hk, d, dtype=torch.bfloat16, device="cuda")
    q, kv = typed(rng, (140, hk, d), "bf16"), typed(rng, (n, hk, d), "bf16")
    k[rows - n:] = kv.cuda()
    out, lse, _ = run(q.cuda(), k, k, [0], [140], [rows - n], [n], "bf16", d ** -0.5)
    compare(q, kv, kv, out, lse, [0], [140], [0], [n], "bf16", d ** -0.5)
    by_head = k.view(hk, rows, d)      # head-major: a head's rows are 77 MB apart from the next one's
    by_head[:, rows - n:] = kv.cuda().transpose(0, 1)
    turned = by_head.transpose(0, 1)
    out, lse, _ = run(q.cuda(), turned, turned, [0], [140], [rows - n], [n], "bf16", d ** -0.5)
    compare(q, kv, kv, out, lse, [0], [140], [0], [n], "bf16", d ** -0.5)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_tiles_of_several_queries_of_one_source(dtype):
    rng = np.random.default_rng(1)
    q, k, v = typed(rng, (600, 4, 64), dtype), typed(rng, (500, 2, 64), dtype), typed(rng, (500, 2, 64), dtype)
    q_start, q_len, k_start, k_len = [0, 300, 430], [290, 130, 170], [3, 3, 110], [390, 390, 333]
    out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), q_start, q_len, k_start, k_len, dtype, 0.125)
    compare(q, k, v, out, lse, q_start, q_len, k_start, k_len, dtype, 0.125)


@gpu
@pytest.mark.parametrize("field,value", [("q_start", -1), ("q_start", 1 << 20), ("q_len", -1), ("q_len", 301), ("k_start", -1),
                                         ("k_start", 3000), ("k_len", 1101), ("k_len", -5), ("k_start", 2147483647)])
@pytest.mark.parametrize("b,heads", [(3, 2), (80, 4)])     # cut into ranges; several waves, the last one cut
def test_long_tiles_leave_bad_lengths_out(field, value, b, heads):
    rng = np.random.default_rng(4)
    q = typed(rng, (300 * b, heads, 32), "bf16").cuda()
    k, v = (typed(rng, (3000, heads, 32), "bf16").cuda() for _ in range(2))
    given = {"q_start": np.arange(b) * 300, "q_len": np.full(b, 300), "k_start": np.arange(b) * 7, "k_len": np.full(b, 1100)}
    good, gl, need = run(q, k, v, *given.values(), "bf16", 0.2, max_q=300, max_k=1100)
    assert status_bits() == 0 and need > 0
    given[field][b - 2] = value
    out, lse, _ = run(q, k, v, *given.values(), "bf16", 0.2, max_q=300, max_k=1100)
    assert status_bits() == 4
    left = torch.zeros(300 * b, dtype=torch.bool, device="cuda")
    left[(b - 2) * 300:(b - 1) * 300] = True
    assert torch.equal(out[~left], good[~left]) and torch.equal(lse[~left], gl[~left])
    assert bool((out[left] == 7).all()) and bool((lse[left] == 7).all())


def test_scales_past_the_largest_power_of_two_are_refused():
    # scores are taken in powers of two: scale * log2(e) has to be a number
    for scale, sound in ((2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False)):
        a = host_args()
        a.scale = scale
        got = L.load().mc_cross_attention(C.byref(a), None)
        assert got == (L.MC_CUDA if sound and not torch.cuda.is_available() else L.MC_INVALID_INPUT)


def test_tensors_of_no_rows_may_be_null():
    lib = L.load()
    a = host_args()
    a.q, a.out, a.q_rows, a.k, a.v, a.k_rows = None, None, 0, None, None, 0
    sound = L.MC_INVALID_INPUT if torch.cuda.is_available() else L.MC_CUDA   # past the checks; there is no such memory
    assert lib.mc_cross_attention(C.byref(a), None) == sound
    for field in ("q_rows", "k_rows"):
        setattr(a, field, 1)
        assert lib.mc_cross_attention(C.byref(a), None) == L.MC_INVALID_INPUT
        setattr(a, field, 0)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-30, 1.5])
@pytest.mark.parametrize("q_len", [1, 150])
def test_scales_of_any_sign(dtype, scale, q_len):
    rng = np.random.default_rng(q_len)
    q, k, v = (typed(rng, (n, 2, 64), dtype) for n in (q_len, 260, 260))
    out, lse, _ = run(q.cuda(), k.cuda(), v.cuda(), [0], [q_len], [0], [260], dtype, scale)
    want, wl = attend(f64(q), f64(k), f64(v), float(np.float32(scale)), np.ones(260, bool))
    dx = 2.0 ** -20 * abs(scale) * np.abs(f64(q)).sum(-1).max() * np.abs(f64(k)).max()
    tol = (2.0 ** -18 if dtype == "f32" else torch.finfo(q.dtype).eps) + 2 * dx
    np.testing.assert_allclose(f64(out), want, rtol=0, atol=tol * np.abs(f64(v)).max())
    np.testing.assert_allclose(f64(lse), wl, rtol=2.0 ** -20, atol=2.0 ** -19 + dx)
