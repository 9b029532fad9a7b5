"""The layers and the clipping from several host threads at once, each on a stream of its own."""
from __future__ import annotations

import threading

import pytest
import torch

import orda_ce_kernel as orda
from tests.test_gpu_layers import ffn_case, linear_case, run_ffn, run_linear

pytestmark = pytest.mark.gpu


def test_threads_give_what_each_gives_alone():
    blocks = [ffn_case(300, 264, 520, 264, torch.bfloat16, "silu", True, seed=s) for s in range(3)]
    layers = [linear_case(90, 97, 77, torch.float16, "gelu", True, True, seed=s) for s in range(3)]
    alone = [(run_ffn(b, "silu"), run_linear(v, "gelu")) for b, v in zip(blocks, layers)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                params = [torch.nn.Parameter(torch.ones(100, device="cuda")) for _ in range(3)]
                for p in params:
                    p.grad = torch.full_like(p, float(i + 1))
                for _ in range(10):
                    got = run_ffn(blocks[i], "silu"), run_linear(layers[i], "gelu")
                    total = orda.clip_grad_norm_(params, 1e9)
                    stream.synchronize()
                    assert all(torch.equal(g[n], a[n]) for g, a in zip(got, alone[i]) for n in a)
                    assert float(total) == pytest.approx((i + 1) * 300 ** 0.5, rel=1e-6)
                with pytest.raises(ValueError, match="x must be"):
                    orda.fused_linear(torch.zeros(3, 8, device="cuda").double(), torch.zeros(4, 8, device="cuda"))
        except BaseException as exc:  # noqa: BLE001  (handed to the test's thread)
            failed.append((i, repr(exc)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
