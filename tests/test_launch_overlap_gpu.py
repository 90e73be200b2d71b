"""Chains of different kernels that share SMs: every launch starts its prologue beside the one before it, and both
hold or ask for tensor memory.  The order that makes this safe is read from the sources on the CPU
(test_tensor_memory_order_cpu.py); here the chains run, and every product keeps the bits it has alone."""
import itertools

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _plans(smb, torch):
    c, gemm = smb.capi, smb.gemm
    g = torch.Generator(device="cuda").manual_seed(4)

    def bf16(m, n, k):
        a, b = (torch.randn(r, k, generator=g, device="cuda").bfloat16() for r in (m, n))
        d = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
        return gemm.Bf16Plan(a, b, d, m, n, k, flags=c.FLAG_OPERANDS_STATIC), d

    def fp4(m, n, k, flags, stages=0):
        ops = []
        for which, rows in ((0, m), (1, n)):
            codes = torch.empty(rows, k // 2, device="cuda", dtype=torch.uint8)
            packed = torch.empty(gemm.sf_packed_bytes(rows, k), device="cuda", dtype=torch.uint8)
            gemm.fill_fp4_device(codes, packed, None, rows, k, 5, which, 0)
            ops += [codes, packed]
        d = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
        plan = gemm.Fp4Plan(*ops, d, m, n, k, flags=flags)
        if stages:
            plan.tune(group_m=stages)
        return plan, d

    def int8(m, n, k):
        a, b = (torch.randint(-127, 128, (r, k), generator=g, device="cuda", dtype=torch.int8) for r in (m, n))
        sa, sb = (torch.rand(r, generator=g, device="cuda") for r in (m, n))
        d = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
        return gemm.I8Plan(a, sa, b, sb, d, m, n, k, flags=c.FLAG_WEIGHTS_STATIC), d

    return [bf16(14080, 128, 512), bf16(8192, 64, 512), fp4(8192, 128, 1024, c.FLAG_OPERANDS_STATIC),
            fp4(16, 4096, 2048, c.FLAG_NONE, 2), fp4(16, 4096, 2048, c.FLAG_DECODE_SINGLE, 2), fp4(64, 2048, 1024, c.FLAG_NONE),
            int8(16, 4096, 2048), int8(100, 1024, 2048), int8(600, 900, 512)]


@pytest.mark.parametrize("streams", [1, 2])
def test_chains_of_kernels_that_share_sms(smb, cuda_device, streams):
    import torch
    plans = _plans(smb, torch)
    assert "resident=2" in plans[0][0].describe() and "resident=2" in plans[1][0].describe()
    alone = []
    for plan, d in plans:
        plan.run()
        plan.check()
        alone.append(d.clone())
    # Every ordered pair once or more, each plan on one stream only (some own a workspace).
    mine = [list(range(i, len(plans), streams)) for i in range(streams)]
    orders = [[i for pair in itertools.product(own, own) for i in pair] for own in mine]
    queues = [torch.cuda.Stream() for _ in range(streams)]

    def chain():
        for i in range(max(map(len, orders))):
            for order, queue in zip(orders, queues):
                plans[order[i % len(order)]][0].run(queue)

    def verify():
        torch.cuda.synchronize()
        for (plan, d), want in zip(plans, alone):
            plan.check()
            np.testing.assert_array_equal(d.view(torch.int16).cpu().numpy(), want.view(torch.int16).cpu().numpy())
            d.zero_()
        torch.cuda.synchronize()

    for _, d in plans:
        d.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        chain()
    verify()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=queues[0]):
        for i in orders[0]:
            plans[i][0].run(queues[0])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for i in mine[0]:
        np.testing.assert_array_equal(plans[i][1].view(torch.int16).cpu().numpy(), alone[i].view(torch.int16).cpu().numpy())
    del graph
    for plan, _ in plans:
        plan.check()
