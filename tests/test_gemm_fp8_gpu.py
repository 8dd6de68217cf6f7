"""Block-scaled fp8 on the GPU: the quantisers and the product, each against a
plain 64-bit statement.

Tolerances.  One rounding to a type t is off by at most eps(t) / 2 of the
value: bf16 2^-8, fp32 2^-24, e4m3 2^-4 (and half of its smallest step, 2^-10
of the scale, below the normal range)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U_BF16, U_F32, U_E4M3 = 2.0 ** -8, 2.0 ** -24, 2.0 ** -4


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _g(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _fp8(rows, k, dev, seed, rows_per_scale=1):
    g = _g(dev, seed)
    x = (torch.randn(rows, k, generator=g, device=dev) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.exp2(torch.rand(-(-rows // rows_per_scale), -(-k // 128), generator=g, device=dev) * 6 - 10)
    return x, s


def _check_quantised(q, scale, x, slack, rows=1):
    """``q`` [R, K] and ``scale`` hold ``x`` (fp64), known to within ``slack`` (fp64)."""
    from connex_b200.ops import reference as R
    want = R.fp8_block_scale(x, rows)
    room = R.fp8_block_scale(slack, rows) + 3 * U_F32 * want
    assert ((scale.double() - want).abs() <= room).all()
    full = (scale.double().repeat_interleave(rows, 0)[:x.shape[0]]).repeat_interleave(128, 1)[:, :x.shape[1]]
    got = q.double() * full
    tol = (U_E4M3 * x.abs()).maximum(2.0 ** -10 * full) * (1 + 2.0 ** -10) + 4 * U_F32 * x.abs() + 2 * slack
    assert ((got - x).abs() <= tol).all()


SHAPES = [(1, 16), (1, 128), (3, 272), (5, 2048), (64, 4096), (130, 1040), (33, 14336), (2000, 144)]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda v: f"{v[0]}x{v[1]}")
def test_quantize(dev, shape, norm):
    from connex_b200 import ops
    T, K = shape
    g = _g(dev, 1)
    wide = torch.randn(T, K + 24, generator=g, device=dev) * torch.exp2(torch.rand(K + 24, generator=g, device=dev) * 8 - 4)
    x = wide.to(torch.bfloat16)[:, 8:8 + K]                  # rows of a wider tensor
    w = (torch.rand(K, generator=g, device=dev) + 0.5).to(torch.bfloat16) if norm else None
    q, scale = ops.quantize_fp8(x, norm=w, eps=1e-5)
    torch.cuda.synchronize()
    assert q.shape == (T, K) and scale.shape == (T, -(-K // 128))
    ref, slack = x.double(), torch.zeros(T, K, dtype=torch.float64, device=dev)
    if norm:
        ref = ref * torch.rsqrt(ref.square().mean(-1, keepdim=True) + 1e-5) * w.double()
        # the sum of squares: products and at most 64 + 5 + 8 additions of a chain, half of that in the root; rsqrtf
        # 2 ulp; two products
        slack = ref.abs() * (40 + 4 + 2) * U_F32
    _check_quantised(q, scale, ref, slack)


@pytest.mark.parametrize("shape", [(8, 16), (128, 128), (72, 400), (384, 512), (1000, 1040)], ids=lambda v: f"{v[0]}x{v[1]}")
def test_quantize_weight(dev, shape):
    from connex_b200 import ops
    N, K = shape
    g = _g(dev, 2)
    w = (torch.randn(N, K, generator=g, device=dev) * torch.exp2(torch.rand(N, 1, generator=g, device=dev) * 6 - 8)).to(torch.bfloat16)
    q, scale = ops.quantize_weight_fp8(w)
    torch.cuda.synchronize()
    assert scale.shape == (-(-N // 128), -(-K // 128))
    _check_quantised(q, scale, w.double(), torch.zeros_like(w, dtype=torch.float64), 128)


def test_quantize_special_values(dev):
    """NaN and infinities become NaN and leave the scale to the others; zeros and tiny numbers take the least one."""
    from connex_b200 import ops
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=dev)
    x[0, :128] = 3.0
    x[0, 0], x[0, 1], x[0, 2] = float("inf"), float("nan"), float("-inf")
    x[1, 130] = 2.0 ** -120
    x[2] = torch.finfo(torch.bfloat16).max
    x[3, :128] = float("nan")
    for q, s in (ops.quantize_fp8(x), ops.quantize_weight_fp8(x[:1])):
        f = q.float()
        assert torch.isnan(f[0, :3]).all() and (f[0, 3:128] == 448).all() and s[0, 0] == torch.tensor(3.0) / 448
        assert (f[0, 128:] == 0).all() and float(s[0, 1]) == pytest.approx(2.0 ** -100 / 448, rel=1e-6)
    q, s = ops.quantize_fp8(x)
    assert float(s[1, 1]) == pytest.approx(2.0 ** -100 / 448, rel=1e-6) and not q[1].float().any()
    assert (q[2].float() == 448).all() and torch.isfinite(s).all()
    assert torch.isnan(q[3, :128].float()).all() and not q[3, 128:].float().any()


def _product_tolerance(a, sa, b, sb):
    """The sums of a block (fp32, 128 products) and of the blocks with their scales: a chain of 128 + nk additions and
    two products, each rounding at most 2^-23 of the sum of magnitudes (the tensor core may truncate)."""
    from connex_b200.ops import reference as R
    mag = R.gemm_fp8(a.float().abs(), sa.abs(), b.float().abs(), sb.abs())
    return mag * (128 + sa.shape[1] + 4) * 2.0 ** -23


GEMMS = [(1, 8, 16), (1, 6144, 1024), (2, 128, 128), (17, 264, 144), (64, 1000, 112), (128, 256, 256), (129, 72, 1040),
         (300, 520, 2048), (513, 1288, 272), (640, 2304, 4096), (16, 4096, 14336), (200, 384, 7168),
         (2300, 4872, 400), (8200, 1096, 1024), (130, 20000, 64), (33, 40, 14336), (1, 128256, 256)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", GEMMS, ids=lambda v: "x".join(map(str, v)))
def test_gemm(dev, shape, residual):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    M, N, K = shape
    a, sa = _fp8(M, K, dev, 11)
    b, sb = _fp8(N, K, dev, 12, 128)
    x = torch.randn(M, N, generator=_g(dev, 13), device=dev).to(torch.bfloat16) if residual else None
    ref = R.gemm_fp8(a, sa, b, sb, x)
    st = ops.new_status(dev)
    out = ops.gemm_fp8(a, sa, b, sb, residual=x, status=st)
    torch.cuda.synchronize()
    ops.check_status(st, "gemm_fp8")
    tol = U_BF16 * ref.abs() + 2 * _product_tolerance(a, sa, b, sb)
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())
    # scales that lie column by column, as the quantiser leaves them; the residual in place; the same bits
    again = x.clone() if residual else torch.full_like(out, 7.0)
    ops.gemm_fp8(a, sa.t().contiguous().t(), b, sb.t().contiguous().t(), out=again, residual=again if residual else None)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("shape", [(1, 256, 128), (5, 512, 400), (64, 2048, 1024), (129, 768, 2064), (700, 2560, 512), (256, 1024, 4096),
                                   (17, 256, 8192), (2200, 5120, 272), (40, 28672, 256)],
                         ids=lambda v: "x".join(map(str, v)))
def test_gemm_silu_mul(dev, shape):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    M, N, K = shape
    a, sa = _fp8(M, K, dev, 21)
    b, sb = _fp8(N, K, dev, 22, 128)
    y = R.gemm_fp8(a, sa, b, sb)
    e = 2 * _product_tolerance(a, sa, b, sb)
    gate, up = (t.flatten(1) for t in y.unflatten(1, (-1, 2, 128)).unbind(2))
    eg, eu = (t.flatten(1) for t in e.unflatten(1, (-1, 2, 128)).unbind(2))
    ref = R.silu_mul_columns(y)
    # SiLU's slope is at most 1.1; the exponential, the quotient and the products 2^-20 of the value (an argument of
    # up to 2^7 in the exponential: 2^-24 of it each)
    slack = 1.1 * eg * (up.abs() + eu) + torch.nn.functional.silu(gate).abs() * eu + 2.0 ** -16 * ref.abs()
    st = ops.new_status(dev)
    q, scale = ops.gemm_fp8(a, sa, b, sb, silu_mul=True, status=st)
    out = torch.empty(M, N // 2, dtype=torch.bfloat16, device=dev)
    assert ops.gemm_fp8(a, sa, b, sb, out=out, silu_mul=True, status=st) is out
    torch.cuda.synchronize()
    ops.check_status(st, "gemm_fp8")
    assert ((out.double() - ref).abs() <= U_BF16 * ref.abs() + slack).all()
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (M, -(-N // 256))
    _check_quantised(q, scale, ref, slack)


def test_gemm_rows_apart(dev):
    """Operands and outputs that are parts of wider tensors; what lies around the output stays."""
    from connex_b200 import ops
    M, N, K = 70, 136, 272
    a, sa = _fp8(M, K, dev, 31)
    b, sb = _fp8(N, K, dev, 32, 128)
    want = ops.gemm_fp8(a, sa, b, sb)
    wide_a = torch.zeros(M, K + 48, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    wide_a.view(torch.uint8)[:, 16:16 + K] = a.view(torch.uint8)
    wide_b = torch.zeros(N + 3, K + 16, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    wide_b.view(torch.uint8)[3:, :K] = b.view(torch.uint8)
    sc = torch.full((4, 3 * M), 1e30, device=dev)
    sc[:3, ::3] = sa.t()
    buf = torch.full((M + 2, N + 16), 7.0, dtype=torch.bfloat16, device=dev)
    ops.gemm_fp8(wide_a[:, 16:16 + K], sc[:3, ::3].t(), wide_b[3:, :K], sb, out=buf[1:-1, 8:-8])
    assert torch.equal(buf[1:-1, 8:-8], want)
    assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, :8] == 7).all() and (buf[:, -8:] == 7).all()


def test_gemm_nan(dev):
    """A NaN in a row of a, or of b, reaches that row or column and no other."""
    from connex_b200 import ops
    M, N, K = 130, 264, 400
    a, sa = _fp8(M, K, dev, 41)
    b, sb = _fp8(N, K, dev, 42, 128)
    a.view(torch.uint8)[129, 399] = 0x7F
    b.view(torch.uint8)[3, 0] = 0xFF
    bad = torch.isnan(ops.gemm_fp8(a, sa, b, sb).float())
    assert bad[129].all() and bad[:, 3].all() and int(bad.sum()) == N + M - 1


def test_empty_calls(dev):
    from connex_b200 import ops
    a, sa = _fp8(3, 256, dev, 51)
    b, sb = _fp8(256, 256, dev, 52, 128)
    assert ops.gemm_fp8(a[:0], sa[:0], b, sb).shape == (0, 256)
    q, s = ops.gemm_fp8(a[:0], sa[:0], b, sb, silu_mul=True)
    assert q.shape == (0, 128) and s.shape == (0, 1)
    q, s = ops.quantize_fp8(torch.empty(0, 256, dtype=torch.bfloat16, device=dev))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    q, s = ops.quantize_weight_fp8(torch.empty(0, 256, dtype=torch.bfloat16, device=dev))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    assert ops.gemm_fp8(a, sa, b[:0], sb[:0]).shape == (3, 0)


def test_every_way_of_a_product(dev):
    """One call for each choice of tile and of CTAs per tile that the sizes lead to: odd rows, columns that fill no
    block, K that does not divide by the CTAs."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    seen = {}
    for silu in (False, True):
        for m in (1, 2, 15, 17, 30, 33, 50, 65, 100, 129, 250, 500, 1000):
            for n in (256, 1280, 2304, 4096, 6144, 14336, 28672):
                for k in (144, 1040, 2064, 4112, 7184):
                    plan = ops._C.gemm_fp8_plan(m, n, k, 2 if silu else 0, sms)
                    if m * n * k < 2 ** 33:
                        seen.setdefault((silu, plan), (m, n, k))
    assert {p[0] for s, p in seen if not s} == {0, 16, 32, 64, 128} and {p[0] for s, p in seen if s} >= {0, 16}
    for (silu, plan), (M, N, K) in seen.items():
        a, sa = _fp8(M, K, dev, 51)
        b, sb = _fp8(N, K, dev, 52, 128)
        st = ops.new_status(dev)
        if silu:
            out = torch.empty(M, N // 2, dtype=torch.bfloat16, device=dev)
            ops.gemm_fp8(a, sa, b, sb, out=out, silu_mul=True, status=st)
            ref = R.silu_mul_columns(R.gemm_fp8(a, sa, b, sb))
            tol = _product_tolerance(a, sa, b, sb)
            full = R.gemm_fp8(a, sa, b, sb)
            gate, up = full.unflatten(1, (-1, 2, 128)).unbind(2)
            tg, tu = tol.unflatten(1, (-1, 2, 128)).unbind(2)
            # d(silu(g) u): silu's slope is below 1.1, silu itself below |g|; bf16 of the result, 2^-20 for exp and divide
            room = (1.1 * 2 * tg * up.abs() + gate.abs() * 2 * tu + 2.2 * 2 * tg * 2 * tu).flatten(1)
            assert ((out.double() - ref).abs() <= (U_BF16 + 2.0 ** -20) * ref.abs() + room).all(), (plan, M, N, K)
        else:
            ref = R.gemm_fp8(a, sa, b, sb)
            err = (ops.gemm_fp8(a, sa, b, sb, status=st).double() - ref).abs()
            assert (err <= U_BF16 * ref.abs() + 2 * _product_tolerance(a, sa, b, sb)).all(), (plan, M, N, K)
        ops.check_status(st)


def test_shared_memory_is_refused(dev):
    from connex_b200 import ops
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=dev)
    same = x.view(torch.float8_e4m3fn).view(-1)[:4 * 256].view(4, 256)
    with pytest.raises(RuntimeError, match="out overlaps"):
        ops.quantize_fp8(x, out=same)
    with pytest.raises(RuntimeError, match="out overlaps"):
        ops.quantize_weight_fp8(x, out=same)
    a, sa = _fp8(128, 256, dev, 61)
    b, sb = _fp8(512, 256, dev, 62, 128)
    with pytest.raises(RuntimeError, match="out overlaps"):
        ops.gemm_fp8(a, sa, b, sb, out=a, silu_mul=True)
    with pytest.raises(RuntimeError, match="scales overlaps"):
        ops.gemm_fp8(a, sa, b, sb, out_scale=sa, silu_mul=True)
    # two ranges of columns of one tensor are apart
    wide = torch.zeros(128, 512, dtype=torch.float8_e4m3fn, device=dev)
    wide[:, :256] = a
    q, s = ops.gemm_fp8(wide[:, :256], sa, b, sb, out=wide[:, 256:], silu_mul=True)
    r, t = ops.gemm_fp8(a, sa, b, sb, silu_mul=True)
    assert torch.equal(q.contiguous().view(torch.uint8), r.view(torch.uint8)) and torch.equal(s, t)
