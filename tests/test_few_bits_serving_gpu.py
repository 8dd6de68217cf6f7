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
