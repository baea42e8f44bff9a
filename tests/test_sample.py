"""mc_sample against its definition in 64 bits: sorted order, prefix sums and a
running sum by id, on logits with ties, masks, infinities, NaN and the types'
lowest values, for vocabularies of one to 393,216 ids.

Tokens are compared exactly.  The kernel's weights are within 2^-41 of their
value, so a token could differ only where a sum lands within about
vocab * 2^-41 of a border: a chance of 1e-6 or less for all the rows here (the
inputs are fixed).  probs: one f32 rounding (2^-24) plus the weights' error
relative to the drawn one, 2^-41 / w for w down to 2^-20: 2^-20 relative.
"""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from marian_cuda import _lib as L  # noqa: E402

gpu = pytest.mark.gpu
DTYPES = {"f32": (torch.float32, L.MC_F32), "f16": (torch.float16, L.MC_F16), "bf16": (torch.bfloat16, L.MC_BF16)}
LOWEST = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}


def reference(x, t, k, p, m, u):
    """One row: x float64 logits -> (token, prob)."""
    if not t >= 0:
        return -1, 0.0
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    ids = np.lexsort((np.arange(x.size), -x))
    ids = ids[x[ids] > -np.inf]
    if ids.size == 0:
        return -1, 0.0
    if t == 0:
        return int(ids[0]), 1.0
    if 0 < k < ids.size:
        ids = ids[:k]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        d = x[ids[0]] - x[ids]
        w = np.where(x[ids] == x[ids[0]], 1.0, np.exp(np.where(np.isinf(d), -np.inf, -d / t)))
    w = np.where(w < 2.0 ** -41, np.round(w * 2.0 ** 40) / 2.0 ** 40, w)
    if p < 1:
        n = 1 + int(np.searchsorted(np.cumsum(w), max(p, 0.0) * w.sum()))
        ids, w = ids[:n], w[:n]
    if m > 0:
        keep = w >= min(m, 1.0)
        ids, w = ids[keep], w[keep]
    by_id = np.argsort(ids)
    sums = np.cumsum(w[by_id])
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), ids.size - 1)
    while w[by_id[at]] == 0:
        at -= 1
    return int(ids[by_id[at]]), float(w[by_id[at]] / sums[-1])


def dev(a, dtype):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def sample(x, t=None, k=None, p=None, m=None, u=None, dtype="f32", mask=None, mask_stride=0, probs=True):
    """x: a CUDA tensor [rows, vocab], rows any number of elements apart."""
    lib = L.load()
    rows, vocab = x.shape
    keep = [dev(t, np.float32), dev(k, np.int32), dev(p, np.float32), dev(m, np.float32), dev(u, np.float32),
            dev(mask, np.uint32) if mask is not None else None]
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((rows,), -7.0, device="cuda")
    at = [None if z is None else z.data_ptr() for z in keep]
    a = L.SampleArgs(logits=x.data_ptr(), temperature=at[0], top_k=at[1], top_p=at[2], min_p=at[3], uniform=at[4],
                     candidates=at[5], tokens=tokens.data_ptr(), probs=pr.data_ptr() if probs else None,
                     row_stride=x.stride(0), candidates_stride=mask_stride, dtype=DTYPES[dtype][1], rows=rows,
                     vocab=vocab)
    torch.cuda.synchronize()
    assert lib.mc_sample(C.byref(a), torch.cuda.current_stream().cuda_stream) == L.MC_OK
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), pr.cpu().numpy().astype(np.float64)


def status_bits():
    bits = C.c_uint32(0)
    assert L.load().mc_op_status(C.byref(bits)) == L.MC_OK
    return bits.value


def check(x, t, k, p, m, u, dtype="f32", **kw):
    xt = x if isinstance(x, torch.Tensor) else torch.from_numpy(np.asarray(x, np.float32)).to(DTYPES[dtype][0]).cuda()
    tokens, probs = sample(xt, t, k, p, m, u, dtype, **kw)
    rows = xt.shape[0]
    x64 = xt.float().cpu().numpy().astype(np.float64)
    f = lambda a, d: np.full(rows, d) if a is None else np.asarray(a, np.float32).astype(np.float64)  # noqa: E731
    t, p, m, u = f(t, 1.0), f(p, 1.0), f(m, 0.0), f(u, 0.0)
    k = np.zeros(rows, int) if k is None else np.asarray(k)
    for i in range(rows):
        token, prob = reference(x64[i], t[i], int(k[i]), p[i], m[i], u[i])
        assert tokens[i] == token, (i, tokens[i], token, t[i], k[i], p[i], m[i], u[i])
        assert probs[i] == pytest.approx(prob, rel=2.0 ** -20, abs=0)
    return tokens


# ---- refusals ---------------------------------------------------------------------

def host_args():
    return L.SampleArgs(logits=1 << 20, temperature=64, top_k=64, top_p=64, min_p=64, uniform=64, tokens=64, probs=64,
                        row_stride=100, dtype=L.MC_F32, rows=2, vocab=100)


@pytest.mark.parametrize("field,value", [("logits", 0), ("logits", (1 << 20) + 2), ("uniform", 0), ("tokens", 0),
                                         ("tokens", 66), ("probs", 65), ("temperature", 3), ("top_k", 2),
                                         ("candidates", 2), ("row_stride", -1), ("dtype", 3), ("dtype", -1),
                                         ("rows", -1), ("rows", 1 << 25), ("vocab", 0), ("vocab", 393217)])
def test_bad_arguments_are_refused(field, value):
    a = host_args()
    setattr(a, field, value)
    assert L.load().mc_sample(C.byref(a), None) == L.MC_INVALID_INPUT


def test_null_and_empty_calls():
    lib = L.load()
    assert lib.mc_sample(None, None) == L.MC_INVALID_INPUT
    a = host_args()
    a.rows = 0
    assert lib.mc_sample(C.byref(a), None) == L.MC_OK
    a = host_args()
    a.candidates, a.candidates_stride = 64, -1
    assert lib.mc_sample(C.byref(a), None) == L.MC_INVALID_INPUT
    if not torch.cuda.is_available():
        assert lib.mc_sample(C.byref(host_args()), None) == L.MC_CUDA


@gpu
def test_host_memory_is_refused():
    host = torch.zeros(1000)
    a = host_args()
    a.logits = host.data_ptr()
    assert L.load().mc_sample(C.byref(a), None) == L.MC_INVALID_INPUT


# ---- the definition ----------------------------------------------------------------

def settings(rng, rows):
    return dict(t=np.where(rng.random(rows) < 0.1, 0.0, rng.uniform(0.3, 2.0, rows)),
                k=np.where(rng.random(rows) < 0.5, rng.integers(1, 300, rows), 0),
                p=np.where(rng.random(rows) < 0.6, rng.uniform(0.05, 1.0, rows), 1.0),
                m=np.where(rng.random(rows) < 0.3, rng.uniform(0.001, 0.3, rows), 0.0), u=rng.random(rows, np.float32))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (4, 33), (7, 1000), (3, 2047), (3, 8193), (40, 32000),
                                        (2, 32001), (3, 100003), (1, 393216)])
def test_mixed_settings(dtype, rows, vocab):
    rng = np.random.default_rng(rows * 7 + vocab)
    x = rng.standard_normal((rows, vocab)) * 2.0 + 9.0 * rng.random((rows, vocab)) ** 200
    check(x, dtype=dtype, **settings(rng, rows))
    assert status_bits() == 0


@gpu
@pytest.mark.parametrize("cluster_rows", [1, 80])
@pytest.mark.parametrize("mode", ["plain", "top_k", "top_p", "min_p"])
def test_one_setting_at_a_time(mode, cluster_rows):
    rng = np.random.default_rng(3)
    rows, vocab = cluster_rows, 32000
    x = rng.standard_normal((rows, vocab)) * 1.5
    u = rng.random(rows, np.float32)
    arg = {"plain": {}, "top_k": {"k": rng.integers(1, vocab + 5, rows)}, "top_p": {"p": rng.uniform(0.01, 0.999, rows)},
           "min_p": {"m": rng.uniform(1e-4, 0.9, rows)}}[mode]
    full = dict(t=None, k=None, p=None, m=None, u=u)
    check(x, **{**full, **arg})


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_ties_go_by_id(dtype):
    rng = np.random.default_rng(5)
    rows, vocab = 24, 5000
    x = np.round(rng.standard_normal((rows, vocab)) * 1.5) * 0.5      # a handful of values, thousands of ties
    x[0] = 1.25                                                       # all equal
    x[1], x[1, 7], x[1, 4000] = -2.0, 3.0, 3.0
    x[2] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)               # -0 and 0 are equal
    x[3] = -1e4
    s = settings(rng, rows)
    s["t"][:4] = [0.7, 0.0, 1.0, 0.5]
    s["k"][0], s["p"][0], s["p"][2] = 17, 0.5, 0.5
    check(x, dtype=dtype, **s)


@gpu
def test_uniform_at_its_ends():
    x = np.zeros((6, 10))
    u = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, -3.0, 7.0, np.nan], np.float32)
    assert check(x, None, None, None, None, u).tolist() == [0, 9, 9, 0, 9, 0]
    # the borders of a fair draw: u = i / 8 starts id i
    tokens = check(np.zeros((8, 8)), None, None, None, None, np.arange(8) / 8)
    assert tokens.tolist() == list(range(8))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masked_logits(dtype):
    rng = np.random.default_rng(6)
    rows, vocab = 12, 4099
    x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 2).to(DTYPES[dtype][0])
    x[:, ::3] = -float("inf")
    x[1, 1::2] = LOWEST[dtype]       # the type's lowest value: as good as never drawn, but there
    x[2] = LOWEST[dtype]             # nothing else: uniform
    x[3] = -float("inf")             # nothing to draw
    x[4, 100] = float("nan")
    x[5] = float("nan")              # nothing to draw
    x[6, 11] = x[6, 901] = float("inf")
    x[7, 5], x[7, 6] = float("inf"), float("nan")
    x[8] = -float("inf")
    x[8, 4098] = -5.0                # one token left
    s = settings(rng, rows)
    s["t"][6], s["t"][3], s["t"][5] = 0.8, 1.0, 0.0
    tokens = check(x.cuda(), dtype=dtype, **s)
    assert status_bits() == 1        # the NaN
    assert tokens[3] == -1 and tokens[5] == -1 and tokens[6] in (11, 901) and tokens[7] == 5 and tokens[8] == 4098


@gpu
def test_temperatures_from_zero_to_infinity():
    rng = np.random.default_rng(7)
    t = np.array([0.0, 1e-45, 1e-30, 1e-3, 0.05, 50.0, 1e30, np.inf], np.float32)
    x = np.repeat(rng.standard_normal((1, 3001)) * 3, len(t), 0)
    x[:, 17] = x[:, 2017] = 20.0      # the largest, twice
    u = np.full(len(t), 0.75)
    for p in (None, np.full(len(t), 0.6)):
        for k in (None, np.full(len(t), 700)):
            check(x, t, k, p, None, u)
    assert status_bits() == 0
    tokens, probs = sample(torch.from_numpy(x.astype(np.float32)).cuda()[:3], np.array([-1.0, np.nan, 1.0]), u=u[:3])
    assert tokens[0] == tokens[1] == -1 and probs[0] == probs[1] == 0 and tokens[2] >= 0
    assert status_bits() == 4


@gpu
def test_settings_past_their_ranges():
    rng = np.random.default_rng(8)
    x = rng.standard_normal((10, 2500)) * 2
    k = np.array([-1, 0, 1, 2499, 2500, 2501, 2**31 - 1, -2**31, 3, 3])
    p = np.array([0.0, -1.0, 1.0, 2.0, np.nan, np.inf, 1e-30, 0.999999, -np.inf, 0.5])
    m = np.array([0.0, -1.0, 1.0, 2.0, np.nan, np.inf, 1e-30, 0.5, 0.0, 1e-45])
    u = rng.random(10)
    check(x, None, k, None, None, u)
    check(x, None, None, p, None, u)
    check(x, None, None, None, m, u)
    check(x, None, k, p, m, u)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_odd_alignment(dtype):
    rng = np.random.default_rng(9)
    whole = torch.from_numpy(rng.standard_normal((6, 5001)).astype(np.float32) * 2).to(DTYPES[dtype][0]).cuda()
    for x in (whole[:, 1:5000], whole[::2, 3:4096], whole[:, :4992], whole[:1].expand(4, 5001)):
        rows = x.shape[0]
        check(x, dtype=dtype, **settings(rng, rows))


@gpu
@pytest.mark.parametrize("shared", [True, False])
def test_candidate_bits(shared):
    rng = np.random.default_rng(10)
    rows, vocab = 9, 3333
    words = (vocab + 31) // 32 + 1
    x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)).cuda()
    allowed = rng.random((1 if shared else rows, vocab)) < 0.1
    allowed[0, :] &= ~(np.arange(vocab) == int(x[0].argmax()))
    if not shared:
        allowed[3] = False
    bits = np.zeros((allowed.shape[0], words * 32), bool)
    bits[:, :vocab] = allowed
    mask = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
    s = settings(rng, rows)
    tokens, probs = sample(x, dtype="f32", mask=mask, mask_stride=0 if shared else words, **s)
    for i in range(rows):
        row = np.where(allowed[0 if shared else i], x[i].cpu().numpy().astype(np.float64), -np.inf)
        f = lambda a: float(np.float32(a))  # noqa: E731
        token, prob = reference(row, f(s["t"][i]), int(s["k"][i]), f(s["p"][i]), f(s["m"][i]), f(s["u"][i]))
        assert tokens[i] == token and probs[i] == pytest.approx(prob, rel=2.0 ** -20)
    assert status_bits() == 0


@gpu
def test_optional_outputs_and_settings():
    rng = np.random.default_rng(11)
    x = torch.from_numpy(rng.standard_normal((5, 700)).astype(np.float32)).cuda()
    u = rng.random(5)
    a, probs = sample(x, u=u, probs=False)
    assert (probs == -7).all()
    b, _ = sample(x, t=np.ones(5), k=np.zeros(5), p=np.ones(5), m=np.zeros(5), u=u)
    assert (a == b).all()


@gpu
def test_the_draw_does_not_depend_on_the_launch():
    # one row alone (spread over more CTAs) and among many
    rng = np.random.default_rng(12)
    x = torch.from_numpy(rng.standard_normal((300, 20000)).astype(np.float32) * 1.7).cuda()
    s = settings(rng, 300)
    many, mp = sample(x, **s)
    for i in range(0, 300, 37):
        one, op = sample(x[i:i + 1], **{n: a[i:i + 1] for n, a in s.items()})
        assert one[0] == many[i] and op[0] == mp[i]
    again, _ = sample(x, **s)
    assert (again == many).all()


@gpu
def test_captured_and_replayed_on_new_logits():
    lib, rng = L.load(), np.random.default_rng(13)
    rows, vocab = 20, 32000
    x = torch.zeros(rows, vocab, device="cuda")
    u = torch.zeros(rows, device="cuda")
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    a = L.SampleArgs(logits=x.data_ptr(), uniform=u.data_ptr(), tokens=tokens.data_ptr(), row_stride=vocab,
                     dtype=L.MC_F32, rows=rows, vocab=vocab)
    sample(x, u=np.zeros(rows))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        assert lib.mc_sample(C.byref(a), side.cuda_stream) == L.MC_OK
    for seed in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 2))
        u.copy_(torch.from_numpy(rng.random(rows, np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        want, _ = sample(x, u=u.cpu().numpy())
        assert (tokens.cpu().numpy() == want).all()


@gpu
@pytest.mark.parametrize("top_k", [0, 50])
def test_min_p_of_one_keeps_the_largest(top_k):
    # whatever (largest - largest) / temperature comes out as in double: with
    # largest / temperature rounded, half of the rows lie below 1
    rng = np.random.default_rng(15)
    rows, vocab = 64, 3000
    x = rng.standard_normal((rows, vocab)) * 5 + 10
    x[::3, 40] = x[::3, 2900] = 60.0       # the largest, twice
    x[::5, 1000:1400] = 70.0               # and 400 times
    check(x, rng.uniform(0.3, 2.0, rows), np.full(rows, top_k), None, np.ones(rows), rng.random(rows))
    assert status_bits() == 0


@gpu
def test_infinite_logits_at_an_infinite_temperature():
    rows, vocab = 6, 900
    x = np.repeat(np.random.default_rng(16).standard_normal((1, vocab)), rows, 0)
    x[:, [11, 500, 800]] = np.inf
    t = np.array([np.inf, np.inf, np.inf, 3e37, 3e37, 1.0])
    k, p = np.array([1, 2, 0, 1, 0, 2]), np.array([1.0, 1.0, 0.6, 1.0, 0.2, 1.0])
    tokens, probs = sample(torch.from_numpy(x.astype(np.float32)).cuda(), t, k, p, None, np.full(rows, 0.75))
    assert tokens.tolist() == [11, 500, 500, 11, 11, 500]
    assert probs.tolist() == [1.0, 0.5, 0.5, 1.0, 1.0, 0.5]


@gpu
def test_subnormal_logits_and_temperatures():
    rng = np.random.default_rng(17)
    rows, vocab = 12, 700
    x = (rng.permuted(np.tile(np.arange(vocab), (rows, 1)), axis=1) * -1e-40).astype(np.float32)
    t = np.full(rows, 2e-39, np.float32)
    t[6:] = 3e-38
    u = rng.random(rows)
    check(x, t, None, None, None, u)
    check(x, t, np.full(rows, 9), None, None, u)
    check(x, t, None, np.full(rows, 0.7), None, u)
    check(x, t, None, None, np.full(rows, 0.3), u)
    assert status_bits() == 0


@gpu
@pytest.mark.parametrize("mode", ["plain", "top_k", "top_p", "min_p"])
def test_logits_far_from_zero(mode):
    # neighbouring floats there, at temperatures of a few of their steps: the
    # weights have to come from the differences
    rng = np.random.default_rng(18)
    rows, vocab = 24, 3000
    offset = 2.0 ** rng.integers(4, 100, rows)
    offset[0], offset[1:8] = 2.0 ** 127, -offset[1:8]
    step = np.abs(offset) * 2.0 ** -22
    x = offset[:, None] + step[:, None] * rng.integers(0, 200, (rows, vocab))
    assert (x == x.astype(np.float32)).all()
    arg = {"plain": {}, "top_k": {"k": rng.integers(1, 400, rows)}, "top_p": {"p": rng.uniform(0.1, 0.99, rows)},
           "min_p": {"m": rng.uniform(0.01, 1.0, rows)}}[mode]
    full = dict(t=step * rng.uniform(2.0, 20.0, rows), k=None, p=None, m=None, u=rng.random(rows))
    check(x, **{**full, **arg})
    assert status_bits() == 0
