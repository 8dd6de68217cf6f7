"""Serving with e4m3 projections and the 4-bit cache on the GPU: the ranks of a tensor-parallel group."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


class _Sum:
    """Stands for the all-reduce of a group whose ranks are threads of this process: the host adds their tensors up
    once all have launched theirs."""

    def __init__(self, world):
        self.meet, self.parts = threading.Barrier(world, timeout=60), [None] * world

    def all_reduce(self, rank, t):
        self.parts[rank] = t.clone()
        torch.cuda.synchronize()
        self.meet.wait()
        t.copy_(sum(p.float() for p in self.parts))
        torch.cuda.synchronize()
        self.meet.wait()


def _steps(rt, prompt, before=lambda ids: None):
    """Logits after a chunked prompt and three decode steps."""
    from connex.pp.handover import CX_CTX, REQUEST_IDS
    got, done = [], 0
    for n in (64, 31, 1, 1, 1):
        ids = torch.tensor(prompt[done:done + n], dtype=torch.int32, device=rt.device)
        before(ids)
        td = {"kind": "decode" if n == 1 else "mixed", REQUEST_IDS: ["a"], CX_CTX: [done], "n_new": [n], "n_dec": 0,
              "ids": ids}
        rt.compute(td, [])
        torch.cuda.synchronize()
        got.append(rt.model.logits[0].float().clone())
        done += n
    rt.check_status()
    return torch.stack(got)


def _partial_tolerance(q, s, w):
    """bf16's rounding aside: a block's 128 products and the blocks with their scales, fp32, each rounding at most 2^-23
    of the sum of magnitudes (the tensor core may truncate)."""
    from connex_b200.ops import reference as R
    return 2 * R.gemm_fp8(q.float().abs(), s, w.q.float().abs(), w.scale) * (128 + s.shape[1] + 4) * 2.0 ** -23


def test_tensor_parallel_ranks(dev):
    """Two ranks with e4m3 shards over 4-bit caches: the shards are the whole's codes, and what each rank puts into an
    all-reduce is the product of its own codes, on rank 0 with the residual."""
    from connex_b200.models.llama import LlamaConfig
    from connex_b200.ops import reference as R
    from connex_b200.parallel.tp import TPGroup
    from connex_b200.serve.engine import _make_runtime
    cfg = LlamaConfig.tiny(layers=2)
    prompt = torch.randint(3, 1000, (100,), generator=torch.Generator().manual_seed(7)).tolist()
    whole = _make_runtime(cfg, 0, 2, dev, 32, 2, 128, 128, None, 5, None, "int4", "fp8")
    want = _steps(whole, prompt)
    world, out, errors = 2, [None, None], []
    ring = _Sum(world)

    class Group(TPGroup):
        def begin(self, ids):
            self.x, self.calls = self.rt.weights.embed[ids.long()], 0

        def all_reduce(self, t):
            name, lw = ("attn", "mid")[self.calls & 1], self.rt.weights.layers[self.calls >> 1]
            w = lw.wo if name == "attn" else lw.w2
            q, s = self.rt.model._q8(name, t.shape[0])
            ref = R.gemm_fp8(q, s, w.q, w.scale, self.x if self.rank == 0 else None)
            assert ((t.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + _partial_tolerance(q, s, w)).all(), (name, self.rank)
            ring.all_reduce(self.rank, t)
            self.x, self.calls = t.clone(), self.calls + 1

    def rank(r):
        try:
            tp = Group(r, world)
            tp.rt = rt = _make_runtime(cfg, 0, 2, dev, 32, 2, 128, 128, None, 5, tp, "int4", "fp8")
            for a, b in zip(rt.weights.layers, whole.weights.layers):
                for n, dim in (("wo", 1), ("w2", 1)):
                    a8, b8 = getattr(a, n), getattr(b, n)
                    assert torch.equal(a8.q.view(torch.uint8), b8.q.view(torch.uint8).chunk(world, dim)[r])
                    assert torch.equal(a8.scale, b8.scale.chunk(world, dim)[r])
            out[r] = _steps(rt, prompt, tp.begin)
            assert tp.calls == 4
        except BaseException as e:  # noqa: BLE001 - told by the thread that waits
            errors.append(e)
            ring.meet.abort()
    threads = [threading.Thread(target=rank, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert torch.equal(out[0], out[1])
    # Next to one GPU with the whole: the partial sums' roundings to bf16 tip inputs of products over to other codes.
    # Two roundings of a value to e4m3 differ by sqrt(2 / 3) 2^-4 of it in the mean square at most, a vector's norm
    # goes through the random weights as any other's does, and the eight quantisations add up in squares.
    assert ((out[0] - want).norm(dim=1) <= (8 * 2 / 3) ** 0.5 * 2.0 ** -4 * want.norm(dim=1)).all()


class _Held:
    """The operators that a model calls, each held to its 64-bit statement on the inputs that the model gives it."""

    def __init__(self, monkeypatch):
        from connex_b200 import ops
        self.counts, self.rows = {}, None
        for name in ("quantize_fp8", "gemm_fp8", "rope_cache_int4", "decode_attention_int4", "prefill_attention_paged_int4",
                     "rmsnorm"):
            monkeypatch.setattr(ops, name, self._of(name, getattr(ops, name)))

    def _of(self, name, real):
        def call(*a, **kw):
            self.counts[name] = self.counts.get(name, 0) + 1
            return getattr(self, name)(real, *a, **kw)
        return call

    def quantize_fp8(self, real, x, norm=None, eps=1e-6, out=None, scale=None):
        from tests.test_gemm_fp8_gpu import U_F32, _check_quantised
        got = real(x, norm=norm, eps=eps, out=out, scale=scale)
        ref, slack = x.double(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        if norm is not None:
            ref = ref * torch.rsqrt(ref.square().mean(-1, keepdim=True) + eps) * norm.double()
            slack = ref.abs() * (40 + 4 + 2) * U_F32          # as in the quantiser's own test
        _check_quantised(*got, ref, slack)
        return got

    def gemm_fp8(self, real, a, sa, b, sb, out=None, out_scale=None, residual=None, silu_mul=False, status=None):
        from connex_b200.ops import reference as R
        from tests.test_gemm_fp8_gpu import U_BF16, _check_quantised, _product_tolerance
        y, e = R.gemm_fp8(a, sa, b, sb), 2 * _product_tolerance(a, sa, b, sb)
        added = None if residual is None else residual.double()
        got = real(a, sa, b, sb, out=out, out_scale=out_scale, residual=residual, silu_mul=silu_mul, status=status)
        if silu_mul:
            (gate, up), (eg, eu) = ((t.flatten(1) for t in z.unflatten(1, (-1, 2, 128)).unbind(2)) for z in (y, e))
            ref = R.silu_mul_columns(y)
            slack = 1.1 * eg * (up.abs() + eu) + torch.nn.functional.silu(gate).abs() * eu + 2.0 ** -16 * ref.abs()
            _check_quantised(*got, ref, slack)
        else:
            ref = y if added is None else y + added
            assert ((got.double() - ref).abs() <= U_BF16 * ref.abs() + e).all()
        return got

    def rmsnorm(self, real, x, weight, eps, out=None, residual=None):
        ref = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + eps) * weight.double()
        got = real(x, weight, eps, out=out, residual=residual)
        assert residual is None and ((got.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -16) * ref.abs()).all()
        return got

    def rope_cache_int4(self, real, qkv, pos, cs, hq, hkv, slots, k, v, out=None, status=None, **norms):
        from tests.test_kv_int4_gpu import BS, D, U_BF16, _codes_hold, _turned
        x = qkv.clone().view(qkv.shape[0], hq + 2 * hkv, D)
        got = real(qkv, pos, cs, hq, hkv, slots, k, v, out=out, status=status, **norms)
        ref, slack = _turned(x[:, :hq], pos, cs, None)
        assert ((got.reshape(ref.shape).double() - ref).abs() <= U_BF16 * ref.abs() + 2 * slack).all()
        blk, off = slots // BS, slots % BS
        kr, ks = _turned(x[:, hq:hq + hkv], pos, cs, None)
        _codes_hold(k[blk, :, off], kr, U_BF16 * kr.abs() + 2 * ks)
        _codes_hold(v[blk, :, off], x[:, hq + hkv:].double(), torch.zeros(x[:, hq + hkv:].shape, device=x.device).double())
        return got

    def _attention(self, q, out, k, v, table, ctx, new, hq, *u):
        from connex_b200.ops import reference as R
        from tests.test_kv_int4_gpu import D, _attention_tolerance
        rows = q[:, :hq * D].reshape(-1, hq, D)
        ref, mag = R.paged_attention_int4(rows, k, v, table, ctx, new)
        tol = _attention_tolerance(ref, mag, rows, k, v, table, ctx, new, *u)
        err = (out.view(ref.shape).double() - ref).abs()
        assert (err <= tol).all(), float((err / tol).max())
        assert err.norm() <= 4 * 2.0 ** -8 * ref.norm()

    def decode_attention_int4(self, real, q, k, v, table, lens, hq, ws, out=None, status=None):
        got = real(q, k, v, table, lens, hq, ws, out=out, status=status)
        self._attention(q, got, k, v, table, [int(n) - 1 for n in lens], [1] * len(lens), hq, 2.0 ** -11)
        return got

    def prefill_attention_paged_int4(self, real, q, k, v, table, tiles, hq, hkv, out=None, status=None, n_blocks=None):
        got = real(q, k, v, table, tiles, hq, hkv, out=out, status=status, n_blocks=n_blocks)
        ctx, new = zip(*self.rows)
        self._attention(q, got, k, v, table, ctx, new, hq, 2.0 ** -8, 2.0 ** -8)
        return got


def test_each_call_of_a_model_on_its_own_inputs(dev, monkeypatch):
    """Whole and chunked prompts, decode rows with them and alone: every operator's result is right for the codes, cache
    rows and buffers that the layers really hand it."""
    from connex.pp.handover import CX_CTX, REQUEST_IDS
    from connex_b200.models.llama import LlamaConfig
    from connex_b200.serve.engine import _make_runtime
    rt = _make_runtime(LlamaConfig.tiny(layers=2), 0, 2, dev, 64, 4, 256, 256, None, 11, None, "int4", "fp8")
    held = _Held(monkeypatch)
    ids = torch.randint(3, 1000, (300,), generator=torch.Generator().manual_seed(12)).tolist()
    steps = [("prefill", [("a", 0, 70), ("b", 0, 17)]), ("mixed", [("a", 70, 1), ("c", 0, 33)]),
             ("mixed", [("b", 17, 1), ("a", 71, 1), ("c", 33, 40), ("d", 0, 5)]),
             ("decode", [("a", 72, 1), ("b", 18, 1), ("c", 73, 1), ("d", 5, 1)])]
    for kind, rows in steps:
        n_dec = sum(n == 1 for _, _, n in rows)
        held.rows = [(c, n) for _, c, n in rows[n_dec if kind == "mixed" else 0:]]
        td = {"kind": kind, REQUEST_IDS: [r for r, _, _ in rows], CX_CTX: [c for _, c, _ in rows],
              "n_new": [n for _, _, n in rows], "n_dec": n_dec if kind == "mixed" else 0,
              "ids": torch.tensor(sum((ids[c:c + n] for _, c, n in rows), []), dtype=torch.int32, device=dev)}
        if kind == "mixed":
            # chunks read the tables behind those of the decode rows
            assert [n for _, _, n in rows][:n_dec] == [1] * n_dec
        rt.compute(td, [])
        torch.cuda.synchronize()
    rt.check_status()
    # two layers, four steps: four products a layer, the quantiser behind both norms and behind the attention
    assert held.counts == {"gemm_fp8": 32, "quantize_fp8": 24, "rope_cache_int4": 8, "rmsnorm": 4,
                           "decode_attention_int4": 6, "prefill_attention_paged_int4": 6}
