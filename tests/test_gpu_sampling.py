"""Sampling against a plain statement of its definition in 64 bits: equal tokens everywhere (ties, masks,
infinities, flat and steep rows, vocabularies around every piece and slice), log probabilities within
fp32's rounding; the same tokens alone, in a batch, on streams and in replayed graphs."""
import ctypes

import numpy as np
import pytest
import torch

from rdkv_amd import _lib, sampling
from tests.gpu_util import DEV, record_native, require_gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def oracle(logits, u, T, k, p, min_p):
    """One row in float64: (token, log probability)."""
    x = np.asarray(logits, np.float64)
    ids = np.flatnonzero(x > -np.inf)
    if ids.size == 0:
        return -1, -np.inf
    ids = ids[np.argsort(-x[ids], kind="stable")]
    if not T > 0:
        return int(ids[0]), 0.0
    v = x[ids]
    z = np.zeros(v.size)
    with np.errstate(over="ignore", invalid="ignore"):
        z[v != v[0]] = (v[v != v[0]] - v[0]) / T
    w = np.exp(z)
    n = v.size if k <= 0 else min(int(k), v.size)
    cum = np.cumsum(w[:n])
    stay = n
    if p < 1:
        stay = min(stay, int(np.searchsorted(cum, p * cum[-1], side="left")) + 1)
    stay = min(stay, max(1, int((w >= min_p).sum())))
    cum = cum[:stay]
    i = min(int(np.searchsorted(cum, u * cum[-1], side="right")), int((w[:stay] > 0).sum()) - 1)
    return int(ids[i]), float(z[i] - np.log(cum[-1]))


def check(logits, u, T=1.0, k=0, p=1.0, min_p=0.0, what=""):
    """Runs the rows, with settings per row or shared, and compares; returns the tokens."""
    B = logits.shape[0]

    def run(rows):
        dev = lambda v, t: torch.as_tensor(v, dtype=t)[rows].to(DEV) if np.ndim(v) else v  # noqa: E731
        return sampling.sample_tokens(logits.to(DEV)[rows.to(DEV)], torch.as_tensor(u, dtype=F32)[rows].to(DEV), temperature=dev(T, F32),
                                      top_k=dev(k, torch.int32), top_p=dev(p, F32), min_p=dev(min_p, F32))

    token, logprob = run(torch.arange(B))
    assert token.dtype == torch.int64 and logprob.dtype == F32
    # a few rows and many go different ways: the rows repeated to thirty, and the last ones alone
    for rows in (torch.arange(30) % B, torch.arange(max(0, B - 4), B)):
        again, lp = run(rows)
        assert torch.equal(again, token[rows.to(DEV)]) and torch.equal(lp, logprob[rows.to(DEV)]), f"{what} rows {rows.tolist()}"
    f32 = lambda v: np.broadcast_to(np.asarray(v, np.float32).astype(np.float64), (B,))  # noqa: E731
    T, p, min_p, u = f32(T), f32(p), f32(min_p), f32(u)
    k = np.broadcast_to(k, (B,))
    x = logits.double().numpy()
    for b in range(B):
        tok, lp = oracle(x[b], u[b], T[b], k[b], p[b], min_p[b])
        got, glp = int(token[b]), float(logprob[b])
        assert got == tok, f"{what} row {b}: token {got}, expected {tok} (T {T[b]} k {k[b]} p {p[b]} min_p {min_p[b]} u {u[b]})"
        # one rounding to fp32 of a number formed in 64 bits (2^-20 of it allowed for those)
        assert glp == lp or abs(glp - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -40, f"{what} row {b}: log probability {glp}, expected {lp}"
    return token


def _logits(B, V, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * scale
    x[:, torch.randint(0, V, (min(V, 5),), generator=g)] += 5.0
    return x.to(dtype), torch.rand(B, generator=g).numpy()


def _mixed(B, V, seed):
    r = np.random.default_rng(seed)
    T = np.where(r.random(B) < 0.15, 0.0, r.uniform(0.3, 2.0, B))
    k = np.where(r.random(B) < 0.5, 0, r.integers(1, max(2, min(V + 3, 400)), B)).astype(np.int32)
    p = np.where(r.random(B) < 0.5, 1.0, r.uniform(0.05, 0.999, B))
    m = np.where(r.random(B) < 0.6, 0.0, r.uniform(0.001, 0.6, B))
    return dict(T=T, k=k, p=p, min_p=m)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 255, 1000, 2049, 4097, 8191, 16384, 16385, 32000, 128256])
def test_mixed_settings(V, dtype):
    require_gpu()
    B = 40 if V < 100_000 else 12
    x, u = _logits(B, V, dtype, V)
    check(x, u, **_mixed(B, V, V + 1), what=f"V {V}")


@pytest.mark.gpu
@pytest.mark.parametrize("setting", [dict(), dict(k=1), dict(k=50), dict(p=0.9), dict(min_p=0.05), dict(T=0.0), dict(T=0.01), dict(T=30.0),
                                     dict(k=50, p=0.9, min_p=0.02, T=0.8), dict(p=1e-6), dict(min_p=1.0), dict(k=10 ** 6)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_shared_settings(setting, dtype):
    require_gpu()
    x, u = _logits(16, 20011, dtype, 5)
    u[0], u[1], u[2] = 0.0, 1 - 2.0 ** -24, 0.5
    check(x, u, **setting)


@pytest.mark.gpu
@pytest.mark.parametrize("V,spread", [(5000, 0.0), (200_003, 0.0), (60_000, 1e-6), (60_000, 0.003), (3000, 0.0), (16_000, 1e-6), (65, 0.0)])
def test_flat_rows(V, spread):
    """Many tokens in one bin (all of them equal, or next to it): the further bins over (logit, index)."""
    require_gpu()
    g = torch.Generator().manual_seed(V)
    x = 1.0 + spread * torch.randn(6, V, generator=g)
    u = torch.rand(6, generator=g).numpy()
    for setting in (dict(), dict(k=V // 3), dict(p=0.5), dict(k=V // 2, p=0.25, min_p=0.5), dict(T=50.0, p=0.7)):
        check(x, u, **setting, what=str(setting))
        check(x.to(BF16), u, **setting, what=f"bf16 {setting}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_values_that_occur_very_often(dtype):
    """More occurrences of one value than 16 bits count: of a positive one, a negative one, zeros of both signs, the lowest
    value as a mask; next to rows that stay just below."""
    require_gpu()
    V = 140_003
    g = torch.Generator().manual_seed(77)
    x = torch.randn(8, V, generator=g)
    often = torch.rand(8, V, generator=g) < 0.7
    for row, v in enumerate([2.5, -1.5, 0.0, -0.0, torch.finfo(dtype).min, 0.0]):
        x[row, often[row]] = v
    x[5, ::2] = torch.where(x[5, ::2] == 0, -0.0, x[5, ::2])
    x[6] = 0.25
    x[6, 65535:] = -3.0 - torch.rand(V - 65535, generator=g)
    x[7] = -0.25
    x[7, 65536:] = -3.0 - torch.rand(V - 65536, generator=g)
    u = torch.rand(8, generator=g).numpy()
    for setting in (dict(), dict(T=0.0), dict(k=60_000), dict(p=0.5, T=3.0), dict(k=100_000, p=0.9, min_p=0.1, T=2.0)):
        check(x.to(dtype), u, **setting, what=str(setting))
        check(x.to(dtype), u[::-1].copy(), **setting, what=str(setting))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V", [3001, 20_001])
def test_masks_infinities_and_no_numbers(V, dtype):
    require_gpu()
    x, _ = _logits(14, V, dtype, 8)
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    x[0] = -inf                                   # nothing left
    x[1] = nan
    x[2, 1:] = -inf                               # one left
    x[3, :-1] = -inf
    x[4, ::2] = -inf
    x[5, 10:] = low                               # masked by the lowest value
    x[6] = low                                    # all of them: they are equals
    x[7, 5] = inf                                 # infinities leave the others without weight
    x[8, [5, 700, 2999]] = inf
    x[9, ::3] = nan
    x[10, ::3], x[10, 1::3] = nan, -inf
    x[11] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)     # equal numbers of different bits
    x[12] = torch.finfo(dtype).max
    x[13, 4], x[13, 5:] = torch.finfo(dtype).max, low
    u = np.linspace(0.02, 0.97, 14)
    for setting in (dict(), dict(k=3), dict(p=0.6), dict(min_p=0.3), dict(T=0.0), dict(k=40, p=0.8, min_p=0.1),
                    dict(T=1e-30), dict(T=1e30), dict(T=float("inf"))):
        if setting.get("T", 1) == float("inf"):
            x[7, 5] = x[8, 5] = x[8, 700] = x[8, 2999] = 3.0      # (infinity over infinity is no number)
        token = check(x, u, **setting, what=str(setting))
        assert token[:3].tolist() == [-1, -1, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V", [131, 9000, 20_001, 70_001, 140_000])
def test_rows_that_one_value_fills(V, dtype):
    """One value at most places, as a mask leaves it or as the largest of all: it has to count where it has weight (the
    temperature is high, it is the largest, nothing else is left) and in top-k, and may not where it has none."""
    require_gpu()
    g = torch.Generator().manual_seed(V)
    low, inf = torch.finfo(dtype).min, float("inf")
    x = torch.randn(16, V, generator=g)
    fill = torch.rand(16, V, generator=g) < 0.98
    for row, v in enumerate([-inf, low, -1e4, float("nan"), -8.0, 3.0, 9.0, 0.0, -0.0]):
        x[row, fill[row]] = v
    x[9] = torch.where(fill[9], low, -inf)                     # nothing else is left
    x[10] = torch.where(fill[10], torch.tensor(-inf), torch.tensor(low))
    x[11, : V // 2] = low                                      # some wavefronts' value, and another's
    x[11, V // 2:] = -inf
    x[11, V // 3] = 1.0
    x[12] = low
    x[12, V - 1] = x[12, 0] = low / 2
    x[13, fill[13]] = torch.finfo(dtype).max
    x[14] = torch.where(fill[14], 0.0, x[14])
    x[14, ::2] = torch.where(x[14, ::2] == 0, -0.0, x[14, ::2])
    x[15, V // 5:] = low
    u = torch.rand(16, generator=g).numpy()
    big = float(torch.finfo(dtype).max) / 4
    for setting in (dict(), dict(T=0.0), dict(k=40), dict(k=V // 2, T=2.0), dict(p=0.9, min_p=0.05), dict(T=big), dict(k=V - 3, p=0.7, T=big),
                    _mixed(16, V, V)):
        check(x.to(dtype), u, **setting, what=str(setting))


@pytest.mark.gpu
def test_borders_and_ties():
    """Borders that are exact in any arithmetic: equal weights, a share that falls on a token's end."""
    require_gpu()
    x = torch.tensor([[2.0, 5.0, 5.0, 5.0, 5.0, 2.0, -1.0, 5.0]]).repeat(9, 1)
    u = np.array([0.0, 0.25, 0.49999997, 0.5, 0.75, 0.99999994, 0.0, 0.5, 0.999])
    k = np.array([4] * 6 + [2, 2, 2], dtype=np.int32)
    token = check(x, u, k=k)                                      # the four of lowest index, a quarter each
    assert token.tolist() == [1, 2, 2, 3, 4, 4, 1, 2, 2]
    assert check(x[:4], [0.0, 0.6, 0.99, 0.5], k=4, p=0.5).tolist() == [1, 2, 2, 2]
    assert check(x[:2], [0.0, 0.99], T=0.0).tolist() == [1, 1]
    # numbers outside [0, 1) act as its ends
    dev = x[:4].to(DEV)
    odd = torch.tensor([-1.0, 1.0, 2.0, float("nan")], device=DEV)
    assert sampling.sample_tokens(dev, odd, top_k=4)[0].tolist() == [1, 4, 4, 1]


@pytest.mark.gpu
def test_settings_on_the_device_out_of_range():
    require_gpu()
    x, u = _logits(6, 500, F32, 3)
    nan = float("nan")
    t = lambda v, d=F32: torch.tensor(v, dtype=d, device=DEV)  # noqa: E731
    run = lambda **kw: sampling.sample_tokens(x.to(DEV), torch.as_tensor(u, dtype=F32).to(DEV), **kw)[0]  # noqa: E731
    plain, first = run(), run(temperature=0.0)
    assert torch.equal(run(top_p=t([1.5, 2, nan, 1, 9, 1])), plain)
    assert torch.equal(run(min_p=t([-1.0, 0, nan, -5, 0, 0])), plain)
    assert torch.equal(run(top_k=t([0, -1, -7, 500, 501, 2 ** 40], torch.int64)), plain)
    assert torch.equal(run(top_p=t([0.0, -1, -2, 0, 0, 0])), first) and torch.equal(run(min_p=t([1.0, 2, 5, 1, 1, 1])), first)
    assert torch.equal(run(temperature=t([0.0, -1, nan, 0, -5, 0])), first)


@pytest.mark.gpu
def test_a_row_does_not_depend_on_its_batch():
    """Alone, in a small and in a large batch (other slices), from rows of another stride, and twice in a row."""
    require_gpu()
    for dtype, V in ((BF16, 50_001), (F32, 9000)):
        x, u = _logits(300, V, dtype, 11)
        s = _mixed(300, V, 12)
        xd, ud = x.to(DEV), torch.as_tensor(u, dtype=F32).to(DEV)
        d = {n: torch.as_tensor(v).to(DEV) for n, v in s.items()}
        call = lambda rows, u_, i: sampling.sample_tokens(rows, u_, temperature=d["T"][i], top_k=d["k"][i], top_p=d["p"][i], min_p=d["min_p"][i])  # noqa: E731
        token, lp = call(xd, ud, slice(None))
        again, lp2 = call(xd, ud, slice(None))
        assert torch.equal(token, again) and torch.equal(lp, lp2)
        wide = torch.full((300, V + 3), float("nan"), dtype=dtype, device=DEV)
        wide[:, 1:V + 1] = xd
        t3, l3 = call(wide[:, 1:V + 1], ud, slice(None))
        assert torch.equal(token, t3) and torch.equal(lp, l3)
        for i in (0, 7, 299):
            one, lp1 = call(xd[i:i + 1], ud[i:i + 1], slice(i, i + 1))
            assert int(one) == int(token[i]) and float(lp1) == float(lp[i])
        few, _ = call(xd[5:25], ud[5:25], slice(5, 25))
        assert torch.equal(few, token[5:25])


@pytest.mark.gpu
def test_shapes():
    require_gpu()
    x, u = _logits(6, 77, F32, 2)
    xd, ud = x.to(DEV), torch.as_tensor(u, dtype=F32).to(DEV)
    token, lp = sampling.sample_tokens(xd, ud)
    t2, l2 = sampling.sample_tokens(xd.view(2, 3, 77), ud.view(2, 3), temperature=torch.ones(2, 3, device=DEV))
    assert t2.shape == (2, 3) and torch.equal(t2.view(-1), token) and torch.equal(l2.view(-1), lp)
    t0, l0 = sampling.sample_tokens(xd[4], ud[4])
    assert t0.shape == () and int(t0) == int(token[4]) and float(l0) == float(lp[4])
    e, _ = sampling.sample_tokens(xd[:0], ud[:0])
    assert e.shape == (0,)
    same, _ = sampling.sample_tokens(xd[:1].expand(6, 77), ud)           # one row, six numbers
    assert int(same[0]) == int(token[0])
    t3, _ = sampling.sample_tokens(xd.t().contiguous().t(), ud)          # columns apart
    assert torch.equal(t3, token)


@pytest.mark.gpu
def test_draws_follow_the_distribution():
    """Evenly spaced numbers: every token's share of them is its probability, to within two numbers' worth."""
    require_gpu()
    n, V = 4096, 50
    x, _ = _logits(1, V, F32, 21, scale=1.0)
    u = (torch.arange(n, dtype=F32) + 0.5) / n
    token, _ = sampling.sample_tokens(x.expand(n, V).to(DEV), u.to(DEV), temperature=0.7)
    share = torch.bincount(token.cpu(), minlength=V).double() / n
    assert float((share - torch.softmax(x[0].double() / 0.7, 0)).abs().max()) <= 2 / n


@pytest.mark.gpu
@pytest.mark.parametrize("B,V", [(33, 30_000), (5, 30_000), (20, 9000)])
def test_streams_and_graphs(B, V):
    require_gpu()
    x, u = _logits(B, V, F16, 4)
    xd, ud = x.to(DEV), torch.as_tensor(u, dtype=F32).to(DEV)
    kw = dict(temperature=0.9, top_p=0.95, top_k=200, min_p=0.001)
    exp = sampling.sample_tokens(xd, ud, **kw)[0]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [sampling.sample_tokens(xd, ud, **kw)[0] for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, exp) for t in got)
    a, au = xd.clone(), ud.clone()
    graphs = []
    for _ in range(2):                                    # two graphs, replayed side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, sampling.sample_tokens(a, au, **kw)[0]))
    for rep in range(3):
        a.copy_(xd.roll(rep, 1))
        au.copy_(ud.roll(rep))
        eager = sampling.sample_tokens(a, au, **kw)[0]
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, eager) for _, out in graphs), f"replay {rep}"


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5003, 20_003])
def test_advance_matches_sample_tokens_and_moves_the_counters(V):
    require_gpu()
    x, u = _logits(4, V, F16, 6)
    s = sampling.Sampling(temperature=0.8, top_k=100, top_p=0.9, min_p=0.01)
    uniforms = torch.as_tensor(u, dtype=F32).to(DEV)
    token, pos, row = (torch.zeros(1, dtype=torch.int64, device=DEV) for _ in range(3))
    n_new = torch.ones(8, dtype=torch.int32, device=DEV)
    pos.fill_(100)
    for step in range(6):                                  # the last two past the numbers: the last one again
        i = min(step, 3)
        logits = x[step % 4].to(DEV).view(1, 1, -1)
        sampling._sample_advance(logits, token, s, uniforms, pos, row, n_new)
        exp, _ = sampling.sample_tokens(logits.view(1, -1), uniforms[i:i + 1], temperature=0.8, top_k=100, top_p=0.9, min_p=0.01)
        assert int(token) == int(exp) and int(pos) == 101 + step and int(row) == step + 1 and n_new.tolist() == [2 + step] * 8


@pytest.mark.gpu
def test_plain_calls_take_the_native_way(monkeypatch):
    """Plain arguments go through csrc/native.cpp, others through the general path, with the same tokens."""
    require_gpu()
    x, u = _logits(6, 700, F16, 12)
    xd, ud = x.to(DEV), torch.as_tensor(u, dtype=F32).to(DEV)
    T, k = torch.full((6,), 0.7, device=DEV), torch.full((6,), 30, dtype=torch.int32, device=DEV)
    calls = record_native(monkeypatch)
    token, lp = sampling.sample_tokens(xd, ud, temperature=T, top_k=k, top_p=0.9, min_p=0)
    same = sampling.sample_tokens(xd, ud, temperature=T, top_k=30, top_p=0.9)[0]
    assert calls.taken == ["sample_rows"] * 2 and torch.equal(same, token)
    for args, kw in (((xd, ud), dict(temperature=T.double(), top_k=k)), ((xd, ud), dict(temperature=T, top_k=k.long())),
                     ((xd.t().contiguous().t(), ud), dict(temperature=T, top_k=k)), ((xd, torch.stack([ud, ud], 1)[:, 0]), dict(temperature=T, top_k=k))):
        t2, l2 = sampling.sample_tokens(*args, top_p=0.9, **kw)
        assert torch.equal(t2, token) and torch.equal(l2, lp)
    assert len(calls.asked) == 6 and len(calls.taken) == 2


def test_refusals_of_the_c_interface():
    lib = _lib.load()
    one = 1 << 20                    # a pointer that is looked at, never followed
    s = _lib.RdkvSampling(temperature_value=1.0, top_p_value=1.0)
    of = lib.rdkv_sample_workspace_bytes
    need = of(2, 20000, 0)
    assert need == of(2, 20000, 1) == of(2, 16385, 2) > 0 and of(40, 20000, 0) == 20 * need
    assert of(0, 20000, 0) == of(-3, 20000, 0) == of(25, 20000, 1) == of(2, 16384, 0) == of(2, 1, 2) == 0

    def rows(logits=one, stride=20000, n=2, vocab=20000, dt=0, u=one, settings=ctypes.addressof(s), token=one, ws=one, nb=need):
        return lib.rdkv_sample_rows(logits, stride, n, vocab, dt, u, settings, token, None, ws, nb, None)

    for bad in (dict(n=-1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(dt=3), dict(settings=None), dict(logits=None), dict(u=None),
                dict(token=None), dict(stride=-64), dict(logits=one + 1, dt=1), dict(logits=one + 2)):
        assert rows(**bad) == _lib.RDKV_EINVAL, bad
    for bad in (dict(ws=None), dict(nb=need - 1), dict(ws=one + 8)):
        assert rows(**bad) == _lib.RDKV_EWORKSPACE, bad
    assert rows(n=0) == _lib.RDKV_OK

    def advance(n_uniform=4, index=one, counter=one, counts=None, n_counts=0, word=None):
        return lib.rdkv_sample_advance(one, 20000, 0, one, n_uniform, index, ctypes.addressof(s), one, counter, None, counts, n_counts, word,
                                       0, None, 0, None)

    for bad in (dict(n_uniform=0), dict(index=None), dict(n_counts=1025, counts=one), dict(n_counts=1), dict(counter=None, word=one)):
        assert advance(**bad) == _lib.RDKV_EINVAL, bad
    assert advance() == _lib.RDKV_EWORKSPACE


def test_no_cpu_path():
    with pytest.raises(RuntimeError):
        sampling.sample_tokens(torch.zeros(2, 5), torch.zeros(2))


@pytest.mark.gpu
def test_refusals():
    require_gpu()
    x, u = torch.zeros(3, 10, device=DEV), torch.zeros(3, device=DEV)
    for kw in (dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0), dict(top_k=1.5), dict(top_k=1 << 31), dict(temperature=float("nan")),
               dict(top_p=float("nan")), dict(temperature=u[:2]), dict(top_k=u), dict(min_p=u.cpu()), dict(top_k=u > 0)):
        with pytest.raises(AssertionError):
            sampling.sample_tokens(x, u, **kw)
    for a, b in ((x.double(), u), (x, u.double()), (x, u[:2]), (x[:, :0], u)):
        with pytest.raises(AssertionError):
            sampling.sample_tokens(a, b)
    with pytest.raises(RuntimeError):
        sampling.sample_tokens(x, u.cpu())
