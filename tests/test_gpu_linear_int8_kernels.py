"""The 8-bit product where its kernels work in earnest: sizes for which the 256 x 256 and the 128 x 128 tiles and the kernel for few
tokens are chosen, with contractions that go round their rings of stages several times and end inside a stage, on varied data."""
import pytest
import torch

import quant_oracle as qo

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.quantized


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


SIZES = [
    # 256 x 256 tiles (on 256 CUs): a ragged edge on both sides, contractions of 17, 33 and 65 stages
    (4095, 4100, 1040), (2049, 4112, 1072), (1023, 8208, 2064), (4095, 2064, 4112),
    # 128 x 128 tiles: whole contractions of 17 and 13 stages, and one cut into seven
    (300, 4112, 2064), (520, 6160, 1552), (200, 777, 4112),
    # rows without 16-byte pieces
    (300, 4111, 2063), (130, 9000, 2001),
    # few tokens: every number of token and channel tiles, rings that are filled again and again
    (64, 6144, 4096), (63, 4090, 8208), (64, 10240, 1040), (32, 8192, 4096), (30, 8200, 2064), (20, 1000, 8192), (16, 8192, 4096),
    (1, 512, 8192), (33, 6144, 4095), (17, 8200, 2049), (5, 8199, 4095),
]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_sums_are_exact(ops, dev, m, n, k):
    """Factors of -1, 0 and 1: sums that fp16 holds exactly, so that every one has to be right."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(m + n + k)
    x = torch.randint(-1, 2, (m, k), generator=gen, device=dev, dtype=torch.int8)
    w = torch.randint(-1, 2, (n, k), generator=gen, device=dev, dtype=torch.int8)
    one = torch.ones((max(m, n),), device=dev)
    want = x.double() @ w.double().t()
    assert float(want.abs().max()) <= 2048
    got = ops.linear_int8(x, w, one[:m], one[:n], out_dtype=torch.float16)
    assert torch.equal(got.double(), want)
    # ... and of whole bytes in rows with gaps
    x = torch.randint(-128, 128, (m, k + 32), generator=gen, device=dev, dtype=torch.int8)[:, 16:16 + k]
    w = torch.randint(-128, 128, (n, k + 16), generator=gen, device=dev, dtype=torch.int8)[:, :k]
    xs, ws = torch.rand((m,), generator=gen, device=dev) + 0.01, torch.rand((n,), generator=gen, device=dev) * 1e-3 + 1e-5
    bias = torch.randn((n,), generator=gen, device=dev)
    got = ops.linear_int8(x, w, xs, ws, bias=bias, out_dtype=torch.bfloat16).double()
    want, bound = qo.linear(x, w, xs, ws, bias, torch.bfloat16)
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())
