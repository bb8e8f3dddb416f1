"""4-bit weights: the quantizer and the layout bit for bit, the products exactly where every partial sum
is a number of fp32, and within rounding elsewhere; sizes where tiles, groups and rows end short."""
import pytest
import torch

from rdkv_amd import _lib, weight_quant as wq
from tests.gpu_util import DEV, record_native, require_gpu

F16, BF16 = torch.float16, torch.bfloat16


def _round20(s):
    """fp32 to 20 significant bits, as a scale word holds it."""
    return ((s.contiguous().view(torch.int32) + 8) & -16).view(torch.float32)


def _quantize_ref(w, G):
    """The quantizer's expressions in fp32 on the CPU: codes, scales and zero points."""
    N, K = w.shape
    x = torch.nn.functional.pad(w.float(), (0, -K % G)).view(N, -1, G)
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    s = _round20((hi - lo) / 15)
    s = torch.where(s < 2.0 ** -120, torch.ones_like(s), s)
    z = torch.round(-lo / s).clamp(0, 15)
    q = (torch.round(x / s[..., None]) + z[..., None]).clamp(0, 15)
    return q.view(N, -1)[:, :K], s, z


def _dense64(codes, scale, zero, G):
    at = torch.arange(codes.shape[1]) // G
    return (codes.double() - zero.double()[:, at]) * scale.double()[:, at]


def _integers(N, K, G, seed, dtype=F16):
    """Codes, power-of-two scales and zero points: every product and sum with small integers is exact in fp32."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    n = -(-K // G)
    scale = 2.0 ** torch.randint(-2, 2, (N, n), generator=g)
    zero = torch.randint(0, 16, (N, n), generator=g, dtype=torch.uint8)
    return codes, scale.to(dtype), zero


def _packed(codes, scale, zero, G, dtype):
    return wq.pack_weight(codes.to(DEV), scale.to(DEV), None if zero is None else zero.to(DEV), G, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,G,dtype", [(1, 1, 32, F16), (16, 128, 128, F16), (17, 129, 32, BF16), (5, 31, 64, F16),
                                         (33, 100, 32, BF16), (64, 1000, 128, BF16), (7, 2048, 64, F16)])
def test_quantizer_codes_scales_and_values(N, K, G, dtype):
    require_gpu()
    g = torch.Generator().manual_seed(N * K)
    w = torch.randn(N, K, generator=g).to(dtype)
    w[:, 0] = 0
    if K > G:
        w[0, :G] = 0                         # a group of zeros
        w[-1, G:] = w[-1, G:].abs()          # groups of one sign
    for view in (w.to(DEV), torch.cat([w, w], 1).to(DEV)[:, :K], w.t().contiguous().to(DEV).t()):
        q = wq.quantize_weight(view, G)
        codes, s, z = _quantize_ref(w, G)
        again = _packed(codes.to(torch.uint8), s, z.to(torch.uint8), G, dtype)
        assert torch.equal(q.codes, again.codes) and torch.equal(q.scales, again.scales)
        assert torch.equal(wq.dequantize_weight(q).cpu(), _dense64(codes, s, z, G).to(dtype))
        assert bool((wq.dequantize_weight(q)[:, 0] == 0).all()), "a zero weight stays zero"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("G", [32, 128])
def test_quantizer_codes_of_quotients_between_two_codes(dtype, G):
    """Quotients in the middle of two whole numbers and a hair off it, at small and large scales: the codes are those of the
    correctly rounded division, rounded to even.  A row's range is 15 units, some with another width in the last bits."""
    require_gpu()
    g = torch.Generator().manual_seed(G)
    N, K = 1024, 512
    unit = 2.0 ** torch.randint(-13, 12, (N, 1), generator=g).double()
    if dtype == BF16:
        unit[: N // 2] = 2.0 ** torch.randint(-122, 122, (N // 2, 1), generator=g).double()
    w = torch.randint(-16, 17, (N, K), generator=g).double() / 2
    w[:, ::G], w[:, 1::G] = -7.5, 7.5
    w[1::2] *= 1 + torch.randint(-3, 4, (N // 2, K), generator=g) * torch.finfo(dtype).eps
    w[2::4, 1::G] *= 1 + torch.randint(0, 9, (N // 4, 1), generator=g) * torch.finfo(dtype).eps
    w = (w * unit).to(dtype)
    codes, s, z = _quantize_ref(w, G)
    q = wq.quantize_weight(w.to(DEV), G)
    exp = _packed(codes.to(torch.uint8), s, z.to(torch.uint8), G, dtype)
    assert torch.equal(q.scales, exp.scales) and torch.equal(q.codes, exp.codes)


@pytest.mark.gpu
def test_quantizer_of_values_that_are_no_numbers_and_of_tiny_ones():
    require_gpu()
    w = torch.randn(20, 256, generator=torch.Generator().manual_seed(3)).to(BF16)
    w[3, 5], w[4, 200], w[5, 0] = float("nan"), float("inf"), -float("inf")
    w[6, :128] = 1e-38
    w[7, :128] = torch.finfo(BF16).max
    w[7, 64:128] = torch.finfo(BF16).min      # a range beyond fp32
    d = wq.dequantize_weight(wq.quantize_weight(w.to(DEV), 128)).cpu()
    bad = torch.isnan(d).view(20, 2, 128).all(-1)
    assert bad.nonzero().tolist() == [[3, 0], [4, 1], [5, 0], [7, 0]]
    assert torch.isnan(d).sum() == 4 * 128 and bool((d[6, :128] == 0).all())
    x = torch.ones(2, 256, dtype=BF16, device=DEV)
    y = wq.linear(x, wq.quantize_weight(w.to(DEV), 128))
    assert torch.isnan(y).any(0).nonzero().view(-1).tolist() == [3, 4, 5, 7]


@pytest.mark.gpu
@pytest.mark.parametrize("scale_dtype", [F16, BF16, torch.float32])
def test_pack_keeps_scales_and_default_zero(scale_dtype):
    require_gpu()
    g = torch.Generator().manual_seed(9)
    codes = torch.randint(0, 16, (19, 200), generator=g, dtype=torch.uint8)
    scale = ((torch.rand(19, 4, generator=g) + 0.1) * torch.tensor([1.0, -1.0, 1e-6, 300.0])).to(scale_dtype)
    q = _packed(codes, scale, None, 64, BF16)
    s = _round20(scale.float())
    assert scale_dtype == torch.float32 or torch.equal(s, scale.float())
    exp = _dense64(codes, s, torch.full((19, 4), 8), 64)
    assert torch.equal(wq.dequantize_weight(q).cpu(), exp.to(BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,G", [(1, 1, 32), (16, 128, 128), (15, 40, 32), (17, 136, 64), (100, 1000, 128),
                                   (333, 777, 32), (48, 4096, 128), (4097, 512, 64), (8, 14336, 128), (3, 32768, 32),
                                   (20, 33000, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_products_of_whole_numbers_are_exact(N, K, G, dtype):
    """Codes, zero points and activations are small integers and scales powers of two, so that every partial sum is
    a whole number of quarters below 2^24: whatever the order, the result is the exact one, rounded once."""
    require_gpu()
    codes, scale, zero = _integers(N, K, G, N + K)
    W = _dense64(codes, scale, zero, G)
    q = _packed(codes, scale, zero, G, dtype)
    g = torch.Generator().manual_seed(K)
    bias = torch.randint(-8, 9, (N,), generator=g).to(dtype)
    for M in (1, 2, 15, 16, 17, 33, 70):
        if M * N * K > 40_000_000:
            continue
        x = torch.randint(-2, 3, (M, K), generator=g).to(dtype)
        assert float((x.double().abs() @ (W.abs() + 16 * scale.double().max()).t()).max()) < 2 ** 21
        exp = (x.double() @ W.t() + bias.double()).to(dtype)
        got = wq.linear(x.to(DEV), q, bias.to(DEV))
        assert torch.equal(got.cpu(), exp), f"{M} rows"
        assert torch.equal(wq.linear(x.to(DEV).float(), q, bias.to(DEV)).cpu(), exp), f"{M} fp32 rows"
        wide = torch.full((M, K + 3), float("nan"), dtype=dtype)
        wide[:, 1:K + 1] = x                     # rows of another stride that start off a 16-byte border
        assert torch.equal(wq.linear(wide.to(DEV)[:, 1:K + 1], q, bias.to(DEV)).cpu(), exp), f"{M} strided rows"


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(5, 8209, 264), (16, 24600, 136), (17, 4113, 700), (33, 2100, 1000), (20, 24600, 130),
                                   (40, 24600, 300), (1030, 1500, 260), (2, 8200, 8), (9, 24577, 127)])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_larger_products_of_whole_numbers_are_exact(M, N, K, G, dtype):
    """As above, where one to sixty-four rows share a tile of the weights and tiles end inside the matrix."""
    require_gpu()
    codes, scale, zero = _integers(N, K, G, M + N)
    W = _dense64(codes, scale, zero, G).to(DEV)
    q = _packed(codes, scale, zero, G, dtype)
    g = torch.Generator().manual_seed(M)
    x = torch.randint(-2, 3, (M, K), generator=g).to(dtype).to(DEV)
    bias = torch.randint(-8, 9, (N,), generator=g).to(dtype).to(DEV)
    exp = x.double() @ W.t()
    guard = torch.full((M * N + 4096,), 7.0, dtype=dtype, device=DEV)
    assert torch.equal(wq.linear(x, q), exp.to(dtype))
    assert torch.equal(wq.linear(x.float(), q, bias), (exp + bias.double()).to(dtype))
    wide = torch.full((M, K + 3), float("nan"), dtype=dtype, device=DEV)
    wide[:, 1:K + 1] = x
    assert torch.equal(wq.linear(wide[:, 1:K + 1], q, out=guard[:M * N].view(M, N)), exp.to(dtype))
    assert bool((guard[M * N:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,G,dtype", [(1, 512, 4096, 128, F16), (1, 130, 14336, 64, BF16), (3, 257, 2027, 32, F16),
                                           (16, 100, 4096, 128, BF16), (70, 64, 1000, 64, F16), (129, 48, 512, 32, BF16)])
def test_products_within_rounding(M, N, K, G, dtype):
    """fp32 sums of n terms with partial sums up to S are off by at most n 2^-24 S; here a group's G products of |x| with
    up to 31 units of scale, its two corrections, and the K / G groups and 8 parts after it, all below
    S = 31 s sum|x|; the rounding to the type adds eps / 2 of the result."""
    require_gpu()
    g = torch.Generator().manual_seed(M + N + K)
    w = (torch.randn(N, K, generator=g) * 0.05).to(dtype)
    x = torch.randn(M, K, generator=g)
    x[:, :: max(1, K // 5)] *= 20
    x = x.to(dtype)
    q = wq.quantize_weight(w.to(DEV), G)
    codes, s, z = _quantize_ref(w, G)
    exp = x.double() @ _dense64(codes, s, z, G).t()
    at = torch.arange(K) // G
    S = 31 * (x.double().abs() @ s.double()[:, at].t())
    bound = torch.finfo(dtype).eps / 2 * exp.abs() + (G + 2 + K / G + 8) * 2.0 ** -24 * S
    got = wq.linear(x.to(DEV), q).double().cpu()
    assert bool(((got - exp).abs() <= bound).all())
    # far inside that bound on the whole: the rounding to the type, and a hundredth of what one code more or less makes
    assert float((got - exp).norm() / exp.norm()) <= torch.finfo(dtype).eps / 2 + 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,G,dtype", [(48, 512, 128, F16), (33, 1000, 64, BF16), (16, 4096, 32, F16), (50, 777, 32, BF16),
                                         (20, 14336, 128, F16), (5, 32768, 128, BF16)])
def test_norm_and_silu_rows(N, K, G, dtype):
    require_gpu()
    g = torch.Generator().manual_seed(K)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)
    q = wq.quantize_weight((rnd(N, K) * 0.1).to(DEV), G)
    W = wq.dequantize_weight(q).double().cpu()
    eps = torch.finfo(dtype).eps
    bias = rnd(N)
    pad = torch.zeros(3, dtype=dtype)

    def check(y, row):
        """One rounding of the result; those of the row's elements (eps / 2 at most, 0.2 eps rms, independent) and of the
        dequantized values that it is compared with add up to 0.4 eps |W| |row|: twelve times that."""
        exp = W @ row.double().reshape(-1) + bias.double()
        bound = eps * exp.abs() + 5 * eps * (W.square() @ row.double().reshape(-1).square()).sqrt()
        assert bool(((y.double().cpu().reshape(-1) - exp).abs() <= bound + 1e-6).all())

    for shift in (0, 3):                       # rows at a 16-byte border, and off it
        put = lambda t: torch.cat([pad[:shift], t.reshape(-1)]).to(DEV)[shift:].view(t.shape)
        h, delta, norm, gate, up = rnd(1, 1, K), rnd(1, 1, K), rnd(K), rnd(1, K), rnd(1, K)
        y, r = wq.norm_linear(put(h), put(delta), put(norm), 1e-5, q, bias.to(DEV))
        r64 = (h.float() + delta.float()).to(dtype)
        assert torch.equal(r.cpu(), r64) and y.shape == (1, 1, N)
        check(y, r64.double() * torch.rsqrt(r64.double().pow(2).mean() + 1e-5) * norm.double())
        hd = put(h)
        y, r = wq.norm_linear(hd, None, put(norm), 1e-5, q, bias.to(DEV))
        assert r is hd
        check(y, h.double() * torch.rsqrt(h.double().pow(2).mean() + 1e-5) * norm.double())
        y = wq.silu_linear(put(gate), put(up), q, bias.to(DEV))
        check(y, torch.nn.functional.silu(gate.float()).to(dtype).double() * up.double())


@pytest.mark.gpu
def test_empty_and_odd_calls():
    require_gpu()
    codes, scale, zero = _integers(20, 64, 32, 1)
    q = _packed(codes, scale, zero, 32, F16)
    assert wq.linear(torch.zeros(0, 64, dtype=F16, device=DEV), q).shape == (0, 20)
    assert wq.linear(torch.zeros(2, 0, 64, dtype=F16, device=DEV), q).shape == (2, 0, 20)
    x = torch.randint(-2, 3, (2, 3, 64), generator=torch.Generator().manual_seed(2)).to(F16)
    exp = (x.double() @ _dense64(codes, scale, zero, 32).t()).to(F16)
    assert torch.equal(wq.linear(x.to(DEV), q).cpu(), exp)
    one = x.to(DEV)[0, 0].expand(5, 64)                              # one row, five times
    assert torch.equal(wq.linear(one, q).cpu(), exp[0, :1].expand(5, 20))
    out = torch.empty(2, 3, 20, dtype=F16, device=DEV)
    assert wq.linear(x.to(DEV), q, out=out) is out and torch.equal(out.cpu(), exp)
    square = wq.quantize_weight(torch.eye(64, dtype=F16, device=DEV), 32)
    both = torch.zeros(20, 64, dtype=F16, device=DEV)
    for y in (both[:10], both[5:15]):                                # (whole rows of one buffer, and rows in part)
        with pytest.raises(AssertionError, match="overlap"):
            wq.linear(both[:10], square, out=y)
    assert bool((wq.linear(both[:10], square, out=both[10:]) == 0).all())
    none = wq.quantize_weight(torch.zeros(0, 64, dtype=F16, device=DEV), 32)
    assert wq.linear(x.to(DEV), none).shape == (2, 3, 0) and wq.dequantize_weight(none).shape == (0, 64)


@pytest.mark.gpu
def test_products_on_streams_and_in_graphs():
    """Two streams at once and a captured graph replayed between eager work: equal bits every time."""
    require_gpu()
    g = torch.Generator().manual_seed(5)
    q = wq.quantize_weight((torch.randn(700, 1500, generator=g) * 0.1).to(F16).to(DEV), 64)
    xs = [torch.randn(m, 1500, generator=g).to(F16).to(DEV) for m in (1, 9, 40)]
    exp = [wq.linear(x, q) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([wq.linear(x.float(), q) for x in xs])        # (fp32 rows: through the workspace)
    torch.cuda.synchronize()
    for parts in got:
        assert all(torch.equal(a, b) for a, b in zip(parts, exp))
    inputs = [x.clone() for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [wq.linear(x, q) for x in inputs]
    for rep in range(3):
        for a, x in zip(inputs, xs):
            a.copy_(x * (rep + 1))
        eager = [wq.linear(a, q) for a in inputs]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), f"replay {rep}"


@pytest.mark.gpu
def test_plain_calls_take_the_native_way(monkeypatch):
    """Plain arguments go through csrc/native.cpp, others through the general path, with the same bits."""
    require_gpu()
    g = torch.Generator().manual_seed(8)
    q = wq.quantize_weight((torch.randn(50, 300, generator=g) * 0.1).to(F16).to(DEV), 32)
    rnd = lambda *s: torch.randn(*s, generator=g).to(F16).to(DEV)  # noqa: E731
    x, bias, h, delta, norm, up = rnd(2, 3, 300), rnd(50), rnd(1, 300), rnd(1, 300), rnd(300), rnd(1, 300)
    calls = record_native(monkeypatch)
    y = wq.linear(x, q, bias)
    n, r = wq.norm_linear(h, delta, norm, 1e-5, q, bias)
    s = wq.silu_linear(h, up, q)
    dense = wq.dequantize_weight(q)
    again = wq.quantize_weight(dense, 64)
    assert calls.taken == ["w4_linear", "w4_norm_linear", "w4_silu_linear", "w4_dequantize", "w4_quantize"]
    del calls.taken[3:], calls.asked[3:]
    for view in (dense.t().contiguous().t(), torch.cat([dense[:1], dense])[1:]):       # columns of another stride; rows as they are
        other = wq.quantize_weight(view, 64)
        assert torch.equal(other.codes, again.codes) and torch.equal(other.scales, again.scales) and other.shape == (50, 300)
    assert calls.taken[3:] == ["w4_quantize"] and calls.asked[3:] == ["w4_quantize"] * 2
    del calls.taken[3:], calls.asked[3:]
    general = wq.linear(x.transpose(0, 1), q, bias)                   # rows that are no plain view
    assert calls.taken[3:] == [] and calls.asked[3:] == ["w4_linear"] and torch.equal(general, y.transpose(0, 1))
    wide = torch.stack([bias, bias], 1)[:, 0]                         # a bias of another stride
    assert torch.equal(wq.linear(x, q, wide), y) and torch.equal(wq.norm_linear(h, delta, norm, 1e-5, q, wide)[0], n)
    assert torch.equal(wq.silu_linear(h, up, q, torch.zeros_like(wide)), s) and len(calls.taken) == 4
    monkeypatch.setattr(_lib, "native", type("None_", (), {"__getattr__": lambda self, name: lambda *a: None})())
    assert torch.equal(wq.linear(x, q, bias), y) and torch.equal(wq.dequantize_weight(q), dense)
    assert torch.equal(wq.quantize_weight(dense, 64).codes, again.codes)
    n2, r2 = wq.norm_linear(h, delta, norm, 1e-5, q, bias)
    assert torch.equal(n2, n) and torch.equal(r2, r) and torch.equal(wq.silu_linear(h, up, q), s)


def test_refusals_of_the_c_interface():
    """What the library refuses, before any device work."""
    lib = _lib.load()
    one = 1 << 20                    # a pointer that is looked at, never followed
    ok = dict(codes=one, scales=one, x=one, xd=1, xs=64, bias=None, M=2, N=16, K=64, G=32, dt=1, y=one, ys=16, ws=None, wb=0)

    def linear(**kw):
        a = {**ok, **kw}
        return lib.rdkv_w4_linear(a["codes"], a["scales"], a["x"], a["xd"], a["xs"], a["bias"], a["M"], a["N"], a["K"],
                                  a["G"], a["dt"], a["y"], a["ys"], a["ws"], a["wb"], None)

    for bad in (dict(G=48), dict(G=0), dict(dt=0), dict(xd=2), dict(K=0), dict(N=-1), dict(M=-1), dict(codes=None),
                dict(scales=None), dict(x=None), dict(y=None), dict(codes=one + 8), dict(ys=15), dict(M=2_000_000), dict(N=1 << 20, ys=1 << 20, K=1 << 17)):
        assert linear(**bad) == _lib.RDKV_EINVAL, bad
    need = lib.rdkv_w4_linear_workspace_bytes
    for bad in (dict(M=17, xd=0), dict(M=1, K=40000, xd=0), dict(M=2, K=7), dict(M=2, N=8208, ys=8208), dict(ws=one, wb=255),
                dict(M=1000, N=800, ys=800, ws=one, wb=need(1000, 800, 64) - 1), dict(M=17, xd=0, ws=one + 8, wb=1 << 20)):
        assert linear(**{**bad, "xs": 1 << 16}) == _lib.RDKV_EWORKSPACE, bad
    assert linear(M=0) == _lib.RDKV_OK and linear(N=0) == _lib.RDKV_OK
    assert lib.rdkv_w4_linear_norm(one, one, one, one, one, 0.0, one, None, 16, 64, 32, 1, one, None) == _lib.RDKV_EINVAL
    assert b"alias" in lib.rdkv_last_error()
    assert lib.rdkv_w4_linear_norm(one, one, one, None, one, 0.0, None, None, 16, 32769, 32, 1, one, None) == _lib.RDKV_EINVAL
    assert lib.rdkv_w4_linear_silu(one, one, one, None, None, 16, 64, 32, 1, one, None) == _lib.RDKV_EINVAL
    assert lib.rdkv_w4_quantize(one, 63, 2, 64, 32, 1, one, one, None) == _lib.RDKV_EINVAL
    assert lib.rdkv_w4_quantize(one, 64, 2, 64, 32, 0, one, one, None) == _lib.RDKV_EINVAL
    assert lib.rdkv_w4_pack(one, 64, one, 3, 2, None, 0, 2, 64, 32, one, one, None) == _lib.RDKV_EINVAL
    assert lib.rdkv_w4_dequant(one, one, 2, 64, 32, 1, one, 63, None) == _lib.RDKV_EINVAL
    assert lib.rdkv_w4_codes_bytes(17, 129) == 4 * 1024 and lib.rdkv_w4_scale_words(17, 129, 32) == 4 * 64
    assert lib.rdkv_w4_codes_bytes(-1, 5) == 0 and lib.rdkv_w4_scale_words(5, 5, 5) == 0
    assert need(0, 9, 64) == need(9, 0, 64) == need(1, 9, 32768) == 0 and need(1, 16, 32769) == 32776 * 2
    assert need(2, 16, 7) == 2 * 8 * 2 and need(16, 8192, 129) == 16 * 136 * 2
    assert need(16, 8208, 8192) == 64 * (4096 + 256) and need(17, 8192, 129) == 2 * (8192 + 512)
    assert need(65, 8192, 128) == 2 * (16384 + 1024)


def test_no_cpu_path():
    w = torch.zeros(4, 64, dtype=F16)
    with pytest.raises(RuntimeError):
        wq.quantize_weight(w)
    with pytest.raises(RuntimeError):
        wq.pack_weight(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1, dtype=F16))


@pytest.mark.gpu
def test_refusals():
    require_gpu()
    w = torch.zeros(4, 64, dtype=F16, device=DEV)
    q = wq.quantize_weight(w, 32)
    x = torch.zeros(2, 64, dtype=F16, device=DEV)
    for call in (lambda: wq.quantize_weight(w, 16), lambda: wq.quantize_weight(w.float()), lambda: wq.quantize_weight(w[0]),
                 lambda: wq.linear(x[:, :63], q), lambda: wq.linear(x.to(BF16), q), lambda: wq.linear(x, q, x[0, :4].float()),
                 lambda: wq.linear(x, q, x[0, :3]), lambda: wq.linear(x, q, out=x), lambda: wq.norm_linear(x, None, x[0], 1e-5, q),
                 lambda: wq.silu_linear(x[:1], x[:1].float(), q), lambda: wq.dequantize_weight(q, x),
                 lambda: wq.pack_weight(x.to(torch.uint8), x[:, :3], None, 32),
                 lambda: wq.pack_weight(x.to(torch.uint8), x[:, :2], x[:, :2], 32)):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(RuntimeError):
        wq.linear(x.cpu(), q)
