"""GPU: every digit of x counts in the few-token products (dense, gated, experts; expanded by the product
kernel itself or before it).  The bounds of test_gpu_gemv.py grow with K and would let the last digits go.

Notation: x is written under a power of two s for 16 elements as s (q_1 + q_2 / 8 + ... + q_8 / 8^7), with digits
q_j of halves from -2 to 1.5; s is the smallest power of two with a largest magnitude of at most 1.5 s.
"""
import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib
from nvfp4_b200 import build as B
from nvfp4_b200 import gemv as V
from nvfp4_b200 import moe
from test_gpu_gemv import TYPES, raw_weights

pytestmark = pytest.mark.gpu
S = 8.0                                   # s of every block: each has one element of 1.5 s
K, N = 512, 200


@pytest.fixture(scope="module", autouse=True)
def _ready(cuda_device):
    B.build()
    _lib.load()


def weights(at_largest, seed, l=1):
    """(packed, atoms, dense fp64) with power-of-two scales of 1 and 2: nonzero codes only where x has a block's largest
    element (column 16 b + b % 16 of block b), or only elsewhere."""
    g = torch.Generator("cuda").manual_seed(seed)
    code = torch.randint(0, 16, (l, N, K), generator=g, device="cuda")
    col = torch.arange(K, device="cuda")
    largest = col % 16 == (col // 16) % 16
    code = torch.where(largest, 7, 0).expand(l, N, K) if at_largest else torch.where(largest, 0, code)
    packed = (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8)
    rb = -(-N // 128)
    two = torch.randint(0, 2, (l, rb, K // 64, 32, 4, 4), generator=g, device="cuda")
    atoms = (0x38 + 8 * two).to(torch.uint8)
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")
    scale = (1.0 + two.double()).permute(0, 1, 4, 3, 2, 5).reshape(l, rb * 128, K // 16)[:, :N]
    return packed, atoms, value[code] * scale.repeat_interleave(16, 2)


def rows_of_digit(m, j, dtype, seed):
    """x whose elements, but for each block's largest, have digits j and (from 2 on) j - 1 only: integers from -2^5 to 2^5 - 1
    (digit 1: -2 to 1) of the unit of digit j, s / 2 / 8^(j - 1)."""
    g = torch.Generator("cuda").manual_seed(seed)
    i = torch.randint(-32, 32, (m, K), generator=g, device="cuda") if j > 1 else torch.randint(-2, 2, (m, K), generator=g, device="cuda")
    x = i.double() * (S / 2 / 8.0 ** (j - 1))
    col = torch.arange(K, device="cuda")
    x = torch.where(col % 16 == (col // 16) % 16, 1.5 * S, x)
    assert torch.equal(x.to(TYPES[dtype]).double(), x)
    return x.to(TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m", [1, 2, 5, 16])
@pytest.mark.parametrize("j", range(1, 9))
def test_products_of_a_single_digit_are_exact(j, m, dtype):
    """The largest elements meet zero codes.  What is left are sums of at most 480 products, integers below 2^5 times
    halves up to 12 times scales of 1 and 2: below 2^19 units, exact in fp32 in any order and digit by digit."""
    packed, atoms, dense = weights(False, seed=j)
    w = V.Weights(packed.permute(1, 2, 0), atoms)
    x = rows_of_digit(m, j, dtype, seed=m)
    want = x.double() @ dense[0].T
    assert bool(want.any())
    assert torch.equal(V.gemv(x, w, out_dtype=torch.float32).double(), want)
    # the gate's product reads the largest elements alone: 32 times 1.5 s 6 and more, whose sigmoid is 1 in fp32;
    # then one rounding
    packed1, atoms1, dense1 = weights(True, seed=j + 50)
    gate = x.double() @ dense1[0].T
    assert float(gate.min()) > 100
    got = V.dual_gemv(x, V.Weights(packed1.permute(1, 2, 0), atoms1), w, out_dtype=torch.float32)
    assert torch.equal(got, gate.float() * want.float())
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens", [2, 20])
@pytest.mark.parametrize("j", range(1, 9))
def test_experts_products_of_a_single_digit_are_exact(j, tokens, dtype):
    e, topk = 5, 3
    packed, atoms, dense = weights(False, seed=j, l=e)
    packed1, atoms1, dense1 = weights(True, seed=j + 50, l=e)
    w, w1 = (moe.ExpertWeights(list(zip(p, a))) for p, a in ((packed, atoms), (packed1, atoms1)))
    ids = torch.randint(0, e, (tokens, topk), generator=torch.Generator().manual_seed(j), dtype=torch.int32).cuda()
    x = rows_of_digit(tokens, j, dtype, seed=tokens)
    flat = ids.reshape(-1).long()
    each = x.double().repeat_interleave(topk, 0)[:, :, None]
    want, gate = ((d[flat] @ each)[:, :, 0] for d in (dense, dense1))
    assert torch.equal(moe.gemv(x, ids, w, out_dtype=torch.float32).double(), want)
    assert torch.equal(moe.dual_gemv(x, ids, w1, w, out_dtype=torch.float32), gate.float() * want.float())
    assert _lib.device_status() == 0


def tolerance(wx):
    """For a row with one element x: the digits are off by at most 2^-23 s, s < x / 0.75: 8/3 2^-24 |x|.  Each digit's
    product with w is exact; the seven fused steps that join them round to 2^-24 of at most 16/7 |w| s, each
    eighth part of the one after it: 2^-24 * 16/7 * 8/7 / 0.75 |w x|, less than 3.5 * 2^-24."""
    return np.abs(wx) * (8 / 3 + 3.5) * 2.0 ** -24


@pytest.mark.parametrize("m", [1, 2, 5, 16])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_products_of_one_element_keep_its_digits(m, dtype):
    """Elements of as many random bits as the type has, each by itself: all eight digits at once, for 16-bit types
    exactly (the product of their 11 bits and the weights' 6 fits into fp32)."""
    n, k = 257, 512
    packed, atoms, dense = raw_weights(n, k, seed=m)
    w = V.Weights(packed[0], atoms[0])
    experts = moe.ExpertWeights([(packed[0], atoms[0])])
    ids = torch.zeros(m, dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(m)
    for _ in range(12):
        x = torch.zeros(m, k, device="cuda")
        at = torch.randint(0, k, (m,), generator=g, device="cuda")
        value = torch.randn(m, generator=g, device="cuda", dtype=torch.float64) * 2.0 ** torch.randint(-12, 12, (m,), generator=g, device="cuda")
        x[torch.arange(m), at] = value.float()
        x = x.to(TYPES[dtype])
        want = (x[torch.arange(m), at].double()[:, None] * dense[0][:, at].T).cpu().numpy()
        for got in (V.gemv(x, w, out_dtype=torch.float32), moe.gemv(x, ids, experts, out_dtype=torch.float32)):
            off = np.abs(got.double().cpu().numpy() - want)
            assert (off <= (tolerance(want) if dtype == "fp32" else 0)).all(), float((off / np.abs(want).clip(1e-300)).max())
