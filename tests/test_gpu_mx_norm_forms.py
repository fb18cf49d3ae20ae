"""Every form of stride_amd.mx.norm: one, two or four rows a workgroup (to 256 and 512 rows, and beyond),
each with a row's values in registers over one, two or up to four rounds, or read again."""
import numpy as np
import pytest
import torch

import mx_plain
import test_gpu_mx as plain
from stride_amd import layout, mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def held(t):
    return (t.codes, t.scales) if isinstance(t, mx.Tiles) else (t,)


def case(rows, dim, with_add, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device=DEV)
    h = torch.full(((rows + 15) // 16 * 16, dim), 99.0, device=DEV)
    h[:rows] = 3 * rand(rows, dim) * (1 + 9 * (torch.rand(dim, generator=gen, device=DEV) < 0.01))
    add = layout.lane_tiles(rand(*h.shape).to(torch.bfloat16)) if with_add else None
    return h, add, 1 + 0.2 * rand(dim)


def fresh(rows, dim, bits):
    return plain.marked(rows, dim, 8) if bits == 8 else torch.full(((rows + 15) // 16, dim // 16, 16, 16), 99, dtype=torch.int16, device=DEV)


def same_as_alone(h, add, gain, rows, bits):
    """One call on all rows and one on each tile's: h and the results, and what lies behind the rows."""
    dim = h.shape[1]
    whole, out = layout.lane_tiles(h), fresh(rows, dim, bits)
    parts, outs = whole.clone(), fresh(rows, dim, bits)
    mx.norm(whole, rows, gain, 1e-5, add=add, out=out, bits=bits)
    for t in range(len(parts)):
        part = fresh(16, dim, bits)
        mx.norm(parts[t:t + 1], min(16, rows - 16 * t), gain, 1e-5, add=None if add is None else add[t:t + 1], out=part, bits=bits)
        for a, b in zip(held(outs), held(part)):
            a[t:t + 1] = b
    assert torch.equal(whole.view(torch.int32), parts.view(torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(held(out), held(outs)))
    return whole, out


@pytest.mark.parametrize("rows", [257, 333, 512, 513, 1003])
@pytest.mark.parametrize("dim", [16, 528, 2064, 4112, 8192, 8208, 12304, 17424, 40976])
def test_each_form_has_the_same_bits(rows, dim):
    """Every row as in a call of at most 16, which have a workgroup a row; h and what lies behind the rows
    are as they were without an addition."""
    for with_add in (False, True):
        h, add, gain = case(rows, dim, with_add, rows + dim)
        for bits in (8, 16):
            print("norm forms", rows, dim, with_add, bits, flush=True)
            after, out = same_as_alone(h, add, gain, rows, bits)
            back = layout.untile_lanes(after, len(h))
            assert (back[rows:] == 99).all() and (with_add or torch.equal(back, h))
            if rows % 16:
                tail = [a[-1].reshape(a.shape[1], -1, 16, a.shape[-1])[:, :, rows % 16:] for a in held(out)]
                assert all((a == (0xA5 if bits == 8 else 99)).all() for a in tail)


@pytest.mark.parametrize("rows,dim", [(300, 528), (300, 8192), (300, 12304), (300, 17424), (600, 528), (600, 2064), (600, 8192), (600, 8208)])
def test_rows_that_are_zero_or_not_finite(rows, dim):
    """Infinities, NaN of several payloads, zeros and a sum of squares beyond fp32, in the rows that share a
    workgroup with others: they keep to themselves."""
    h, _, gain = case(rows, dim, False, rows * dim)
    odd = {1: float("inf"), 18: float("-inf"), 35: float("nan"), rows - 1: float("nan")}
    for r, v in odd.items():
        h[r, dim // 2] = v
    bits = torch.tensor([0x7FFFFFFF, -1, 0x7F800001], dtype=torch.int32, device=DEV)
    h.view(torch.int32)[rows - 3, torch.tensor([0, dim // 2, dim - 1], device=DEV)] = bits
    h[4], h[5] = 0, 1e30
    for b in (8, 16):
        print("norm odd rows", rows, dim, b, flush=True)
        _, out = same_as_alone(h, None, gain, rows, b)
        v = (mx.dequantize(out, rows, dtype=torch.float32) if b == 8 else layout.untile_lanes(out, rows).view(torch.bfloat16).float())
        nan = v.isnan()
        for r in (35, rows - 1, rows - 3):
            assert nan[r].all()
        for r in (1, 18):  # an infinite sum: 0 but where 0 meets the infinity
            assert nan[r].any() and (v[r][~nan[r]] == 0).all() and nan[r, dim // 2]
        assert (v[4] == 0).all() and (v[5] == 0).all()
        rest = [r for r in range(rows) if r not in odd and r != rows - 3]
        assert not nan[rest].any()


@pytest.mark.parametrize("with_add", [False, True])
@pytest.mark.parametrize("rows,dim", [(3, 33296), (2, 65536), (259, 528), (259, 2064), (259, 8208), (515, 48), (515, 528), (515, 2064)])
def test_against_64_bits(rows, dim, with_add):
    """Rows of more than 32768 columns, and several rows a workgroup."""
    plain.test_norm(rows, dim, with_add)


@pytest.mark.parametrize("rows,dim", [(1, 16), (2, 48), (5, 512), (17, 528), (3, 17424), (300, 528), (515, 2064)])
def test_results_of_8_and_16_bits_are_of_the_same_values(rows, dim):
    """The live rows, codes and scales, of a call whose h is the former one's sum; and both results round
    the same value, one to half a step of e4m3 (2^-4 of it, or 2^-10 of its scale), the other of bf16
    (2^-8 of it)."""
    print("norm values", rows, dim, flush=True)
    h, add, gain = case(rows, dim, True, rows + 7 * dim)
    ht = layout.lane_tiles(h)
    eight = mx.norm(ht, rows, gain, 1e-5, add=add)
    again = mx.norm(ht, rows, gain, 1e-5)
    half = mx.norm(ht, rows, gain, 1e-5, bits=16)
    (code, byte), other = (mx_plain.unpack(t.codes.cpu().numpy(), t.scales.cpu().numpy(), 8) for t in (eight, again))
    assert np.array_equal(code[:rows], other[0][:rows]) and np.array_equal(byte[:rows], other[1][:rows])
    x = layout.untile_lanes(half.cpu(), rows).view(torch.bfloat16).double().numpy()
    got, scale = mx_plain.decode(code, byte, 8)[:rows, :dim], np.repeat(2.0 ** (byte[:rows] - 127.0), 32, 1)[:, :dim]
    most = np.abs(x) / (1 - 2.0 ** -8)
    assert (np.abs(got - x) <= np.maximum(2.0 ** -4 * most, 2.0 ** -10 * scale) + 2.0 ** -8 * most).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows", [1, 3, 15, 16, 17, 33])
def test_quantize_to_a_fresh_result(rows, bits):
    """The live rows of a result that the call allocates are those of one that was passed."""
    rng = np.random.default_rng(rows + bits)
    src = plain.tiles_of(plain.acts_of(rng, rows, 528), torch.float32)
    passed, made = mx.quantize(src, rows, bits=bits, out=plain.marked(rows, 528, bits)), mx.quantize(src, rows, bits=bits)
    a, b = (mx_plain.unpack(t.codes.cpu().numpy(), t.scales.cpu().numpy(), bits) for t in (passed, made))
    assert a[0].shape[0] >= rows and np.array_equal(a[0][:rows], b[0][:rows]) and np.array_equal(a[1][:rows], b[1][:rows])
    assert (b[0][rows:] == 0).all() and (b[1][rows:] == 0).all()
