"""Waits that run out in the kernels of the operators in few bits, on the GPU: recorded, bounded, and without
consequences for the calls after.  A limit of zero makes them run out."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, BS = 128, 16


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _g(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


@pytest.mark.parametrize("heads", [(32, 8), (16, 1)])
@pytest.mark.parametrize("lens", [[4096] * 48, [20000, 1, 0, 700], [3000, 17] * 40], ids=lambda v: f"{len(v)}x{max(v)}")
def test_decode_whose_copies_are_lost(dev, heads, lens):
    """Their rows read as NaN and the workspace is left ready: the next call with it gives the bits of any other.  The
    first half of each table holds no blocks, so that CTAs that lose nothing share pairs with those that do."""
    from connex_b200 import _C, ops
    from connex_b200.ops import reference as R
    hq, hkv = heads
    B, need = len(lens), [-(-n // BS) for n in lens]
    nb = min(sum(need), 1500)
    k, v = (R.int4_rows(torch.randn(nb, hkv, BS, D, generator=_g(dev, s), device=dev).to(torch.bfloat16)) for s in (1, 2))
    table = torch.randint(0, nb, (B, max(need)), generator=_g(dev, 3), device=dev).to(torch.int32)
    half = table.clone()
    for b, n in enumerate(need):
        half[b, :n // 2] = -1
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = torch.randn(B, hq * D, generator=_g(dev, 4), device=dev).to(torch.bfloat16)
    ws = ops.decode_workspace_int4(B, hq, hkv, dev)
    want = ops.decode_attention_int4(q, k, v, table, lt, hq, ws)
    first = _C.decode_int4_rows(0, 0, hkv, hq // hkv)                     # the counters lie behind the partial results
    for _ in range(3):
        st, out = ops.new_status(dev), torch.zeros_like(want)
        _C.decode_attention_int4(q, k, v, half, lt, out, hq, D ** -0.5, ws, st, wait_ns=0)
        with pytest.raises(RuntimeError, match="timeout|bounds"):
            ops.check_status(st)
        assert not ws[first:].any()
        assert out[lt > 0].isnan().all() and (out[lt == 0] == 0).all()
        st = ops.new_status(dev)
        assert torch.equal(ops.decode_attention_int4(q, k, v, table, lt, hq, ws, status=st), want)
        ops.check_status(st)


@pytest.mark.parametrize("graphs", [False, True])
def test_stepper_raises_what_a_step_recorded(dev, graphs):
    """A status word that a step leaves behind fails that step and no other."""
    from connex_b200.models.llama import LlamaConfig
    from connex_b200.serve.engine import ModelStepper
    st = ModelStepper(LlamaConfig.tiny(), dev, 64, max_batch=4, max_ctx=128, max_step_tokens=128, kv_dtype="int4",
                      weight_dtype="fp8", graphs=graphs)
    seq = list(range(3, 40))
    seq += st.prefill(["a"], [seq])
    want = st.decode(["a"], [seq])
    st.rt.model.status.fill_(1)
    with pytest.raises(RuntimeError, match="timeout"):
        st.decode(["a"], [seq])
    assert st.decode(["a"], [seq]) == want


LATE = [("silu", 300, 5120, 1040), ("silu8", 600, 28672, 512), ("add", 1500, 4096, 2064), ("store", 4000, 5000, 272),
        ("store", 1, 6144, 4096), ("add", 33, 4096, 1040), ("store", 64, 4096, 14336), ("add", 613, 2048, 4096),
        ("silu", 5, 512, 4112), ("silu8", 40, 14336, 2064)]


def _product(dev, epi, M, N, K):
    """(call(out, scale, status, wait_ns), empty outputs) of a block-scaled product."""
    from connex_b200 import _C, ops
    a, sa = ops.quantize_fp8(torch.randn(M, K, generator=_g(dev, 11), device=dev).to(torch.bfloat16))
    b, sb = ops.quantize_weight_fp8(torch.randn(N, K, generator=_g(dev, 12), device=dev).to(torch.bfloat16))
    x = torch.randn(M, N, generator=_g(dev, 13), device=dev).to(torch.bfloat16) if epi == "add" else None
    n = N // 2 if epi.startswith("silu") else N
    code = {"store": ops.EPI_STORE, "add": ops.EPI_ADD}.get(epi, ops.EPI_SILU_MUL)

    def empty():
        out = torch.full((M, n), 7.0, device=dev).to(torch.float8_e4m3fn if epi == "silu8" else torch.bfloat16)
        return out, torch.full((M, n // 128), 7.0, device=dev) if epi == "silu8" else None

    def call(out, scale, status=None, wait_ns=-1):
        _C.gemm_fp8(a, sa, b, sb, out, scale, x, code, status, wait_ns=wait_ns)
    return call, empty


@pytest.mark.parametrize("epi,M,N,K", LATE)
def test_product_whose_operands_are_lost(dev, epi, M, N, K):
    """Where every other CTA loses its operands, the call ends, says so, and each output is right or NaN: of CTAs that
    share a tile, one loses what all add up.  The calls after it are as any other."""
    from connex_b200 import ops
    call, empty = _product(dev, epi, M, N, K)
    want = empty()
    call(*want)
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    _, splits = ops._C.gemm_fp8_plan(M, N, K, 2 if epi.startswith("silu") else 0, sms)
    for _ in range(3):
        st, part = ops.new_status(dev), empty()
        call(*part, st, 0)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="timeout"):
            ops.check_status(st)
        got, right = part[0].float(), want[0].float()
        lost = got.isnan()
        assert lost.all() if splits > 1 else lost.any() and not lost.all()
        assert torch.equal(got[~lost], right[~lost])
        if epi == "silu8":                              # a row's 128 outputs that have a scale are lost together
            blocks = lost.view(M, -1, 128)
            assert torch.equal(blocks.any(-1), blocks.all(-1))
            assert torch.equal(part[1][~blocks.all(-1)], want[1][~blocks.all(-1)])
        st, again = ops.new_status(dev), empty()
        call(*again, st)
        ops.check_status(st)
        for x, y in zip(again, want):
            assert x is y is None or torch.equal(x.float(), y.float())
