"""The int8 product with weights that are as new as the stream allows: the same bits with and without chained launches, eagerly
and replayed from a graph in which the weights are written right before."""

import pytest

from mylocal_llm_b200 import Int8Weight, _lib, int8_linear, int8_matmul, quantize_int8_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (5, 4096, 1000), (100, 256, 4096), (700, 2048, 512)])
@pytest.mark.parametrize("graphed", [False, True])
def test_weights_written_right_before(cuda, monkeypatch, m, n, k, graphed):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(m)
    dense = [torch.randn(n, k, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(4)]
    x = torch.randn(m, k, device="cuda", generator=gen)
    source = torch.empty_like(dense[0])

    def products():
        weight = Int8Weight.quantize(source)                                    # (a copy of the codes where K is no multiple of 16)
        codes, scales = quantize_int8_rows(x)
        fresh = Int8Weight.quantize(source)
        outs = [int8_matmul(codes, scales, weight), int8_matmul(codes, scales, fresh), int8_linear(x, Int8Weight.quantize(source))]
        weight.codes.zero_()
        outs.append(int8_linear(x, weight))                                     # overwritten in place
        weight.codes.copy_(fresh.codes)
        return outs + [int8_linear(x, weight)]

    def run(chain):
        monkeypatch.setenv("B200Q_CHAIN", chain)
        source.copy_(dense[0])
        products()
        torch.cuda.synchronize()
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = products()
        seen = []
        for d in dense * 3:
            source.copy_(d)
            if graphed:
                graph.replay()
            else:
                outs = products()
            seen.append([o.clone() for o in outs])
        torch.cuda.synchronize()
        return seen

    plain, chained = run("0"), run("1")
    for a, b in zip(plain, chained):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2]) and torch.equal(a[0], a[4]) and not a[3].any()
    assert _lib.device_status() == 0
