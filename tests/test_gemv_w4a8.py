"""Few-row W4A8 product: the bits of the CPU oracle and of the large product, its refusals, strides and offsets."""
import pytest
import torch

from k2q import ops
from oracle import convrot_ref as R


def make(m, n, k, seed, device="cuda", bias=True):
    g = torch.Generator().manual_seed(seed)
    xq = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    wq = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)      # every nibble, -8 included
    sx = torch.rand(m, generator=g) * 0.05 + 1e-3
    sw = ((torch.rand(n, k // 128, generator=g) - 0.1) * 0.01).bfloat16()
    b = torch.randn(n, generator=g) if bias else None
    if m > 1:
        xq[1] = 0                                                                # a token of zeros
    sw[0] = 0
    return [None if t is None else t.to(device) for t in (xq, sx, wq, sw, b)]


def same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


SHAPES = [(1, 16, 128), (1, 6144, 256), (2, 48, 384), (3, 144, 1152), (5, 272, 2560), (7, 80, 6144), (8, 32, 4096),
          (9, 112, 640), (13, 64, 16384), (16, 256, 896), (17, 96, 1280), (24, 16, 128), (25, 208, 3328), (32, 1040, 2560),
          (32, 16, 16384), (4, 36864, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_bits_of_the_oracle(m, n, k):
    xq, sx, wq, sw, b = make(m, n, k, 100 + m, bias=n % 32 == 0)
    y = ops.gemv_w4a8(xq, sx, wq, sw, b)
    cpu = [None if t is None else t.cpu() for t in (xq, sx, wq, sw, b)]
    assert same_bits(y.cpu(), R.linear_int4_exact(*cpu))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1024, 2560), (6, 272, 1152), (13, 144, 6144), (32, 528, 640)])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
@pytest.mark.parametrize("rank", [0, 1, 13, 32])
def test_bits_of_the_large_product(m, n, k, act, rank):
    """The rows stand in a batch of 40, which only the large product takes."""
    xq, sx, wq, sw, b = make(40, n, k, 7)
    u = torch.randn(40, rank, device="cuda") if rank else None
    bm = torch.randn(n, rank, device="cuda") * 0.1 if rank else None
    kw = dict(lora_scale=-0.7, act=act) if rank else dict(act=act)
    want = ops.gemm_w4a8(xq, sx, wq, sw, b, u=u, bm=bm, **kw)
    got = ops.gemv_w4a8(xq[:m].contiguous(), sx[:m].contiguous(), wq, sw, b, u=None if u is None else u[:m], bm=bm, **kw)
    assert same_bits(got, want[:m])


@pytest.mark.gpu
def test_gelu_against_64_bits():
    m, n, k = 5, 208, 1024
    xq, sx, wq, sw, b = make(m, n, k, 9)
    y = ops.gemv_w4a8(xq, sx, wq, sw, b, act="gelu_tanh").double()
    q = R.unpack_int4(wq.cpu()).double().cuda().reshape(n, k // 128, 128) * sw.double()[:, :, None]
    v = (xq.double() @ q.reshape(n, k).t()) * sx.double()[:, None] + b.double()
    want = torch.nn.functional.gelu(v, approximate="tanh")
    size = (xq.double().abs() @ q.abs().reshape(n, k).t()) * sx.double()[:, None] + b.double().abs()
    # one bf16 rounding, the hardware tanh's 6e-4 on half the value, one fp32 rounding per group and three more
    # (the activation's slope is below 1.13)
    tol = 2.0 ** -8 * want.abs() + 3e-4 * v.abs() + 1.13 * (k // 128 + 4) * 2.0 ** -24 * size
    assert ((y - want).abs() <= tol).all()


@pytest.mark.gpu
def test_out_strides_empty_streams_graph():
    m, n, k = 3, 80, 512
    xq, sx, wq, sw, b = make(m, n, k, 3)
    want = ops.gemv_w4a8(xq, sx, wq, sw, b)
    wide = torch.full((m, n + 24), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.gemv_w4a8(xq, sx, wq, sw, b, out=wide[:, 9:9 + n])                       # odd offset: rows are not 16-byte aligned
    assert same_bits(wide[:, 9:9 + n].contiguous(), want) and (wide[:, :9] == 5).all() and (wide[:, 9 + n:] == 5).all()
    assert ops.gemv_w4a8(xq[:0], sx[:0], wq, sw, b).shape == (0, n)
    odd = torch.empty(n * (k // 128) + 1, dtype=torch.bfloat16, device="cuda")   # scales at an odd address
    odd[1:] = sw.reshape(-1)
    assert same_bits(ops.gemv_w4a8(xq, sx, wq, odd[1:].view(n, k // 128), b), want)
    one = ops.gemv_w4a8(xq[2:], sx[2:], wq, sw, b)                               # a row alone: the same bits
    assert same_bits(one, want[2:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gemv_w4a8(xq, sx, wq, sw, b)
    side.synchronize()
    assert same_bits(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.gemv_w4a8(xq, sx, wq, sw, b)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert same_bits(got, want)


@pytest.mark.gpu
def test_codes_past_32_bits():
    n, k = 262160, 16384                                                         # 2^31 + 131072 bytes of codes
    g = torch.Generator(device="cuda").manual_seed(4)
    wq = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    sw = (torch.rand(n, k // 128, generator=g, device="cuda") * 0.01).bfloat16()
    xq, sx, _, _, _ = make(2, 16, k, 5, bias=False)
    y = ops.gemv_w4a8(xq, sx, wq, sw)
    for a in (0, n - 32):
        assert same_bits(y[:, a:a + 32].contiguous(), ops.gemv_w4a8(xq, sx, wq[a:a + 32].contiguous(), sw[a:a + 32].contiguous()))


def test_refusals():
    xq, sx, wq, sw, b = make(2, 32, 256, 1, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gemv_w4a8(xq, sx, wq, sw, b)
    good = dict(xq=xq, sx=sx, wq4=wq, sw4=sw, bias=b, u=None, bm=None)
    for bad in (dict(xq=xq.float()), dict(xq=xq[:, :128]), dict(wq4=wq.to(torch.int8)), dict(sw4=sw.float()), dict(sw4=sw[:, :1]),
                dict(sx=sx[:1]), dict(sx=sx.double()), dict(bias=b[:5]), dict(u=torch.zeros(2, 4)),
                dict(u=torch.zeros(2, 4), bm=torch.zeros(32, 5)), dict(wq4=wq.t().contiguous().t())):
        with pytest.raises(ValueError):
            ops._check_w4a8("t", **{**good, **bad})
    assert ops._check_w4a8("t", **good) == (2, 32, 256)


@pytest.mark.gpu
def test_refusals_on_gpu():
    xq, sx, wq, sw, b = make(33, 32, 256, 1)
    with pytest.raises(ValueError, match="up to 32"):
        ops.gemv_w4a8(xq, sx, wq, sw, b)
    odd = torch.zeros(2 * 256 + 1, dtype=torch.int8, device="cuda")[1:].view(2, 256)
    with pytest.raises(ValueError, match="aligned"):
        ops.gemv_w4a8(odd, sx[:2].contiguous(), wq, sw, b)
    with pytest.raises(ValueError):
        ops.gemv_w4a8(xq[:2], sx[:2], wq[:24], sw[:24], None)                    # N not a multiple of 16
    with pytest.raises(ValueError):
        ops.gemv_w4a8(xq[:2], sx[:2], wq, sw, b, u=torch.zeros(2, 33, device="cuda"), bm=torch.zeros(32, 33, device="cuda"))


@pytest.mark.gpu
def test_two_host_threads():
    """Calls of very different shared memory needs from two threads at once: a kernel's limit serves both."""
    import threading
    small, large = make(1, 64, 2560, 1), make(8, 64, 16384, 2)            # one kernel, 20 and 200 KB
    want = [ops.gemv_w4a8(*c) for c in (small, large)]
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(2)

    def work(c, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(timeout=30)
                for _ in range(4000):
                    y = ops.gemv_w4a8(*c)
                torch.cuda.current_stream().synchronize()
                assert same_bits(y, w)
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=cw) for cw in zip((small, large), want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
