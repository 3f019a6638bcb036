"""The 4-bit layers on the GPU against their definition in 64 bits.

Tolerances, all derived from the arithmetic. A product's factors are exact and its sums float32: with mag = sum |code x
scale| + sum |bias x| (what the two sums of a group add up), every addition loses at most 2^-23 of mag (the tensor
cores truncate), and a row of c columns in groups of G takes at most 4 c / 32 (two MMA steps a run, in two parts) + 3 c /
G (the group's end) + 40 (warps, CTAs) of them. A result in type t is rounded once more: eps(t) / 2 of its value (and half
the least subnormal, 2^-25, in float16). The SwiGLU kept between the launches is rounded to t once."""

import copy
import ctypes

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from strata_mlx_b200 import _lib, affine, fused  # noqa: E402

F16, F32 = torch.float16, torch.float32


def parts(gen, lead, rows, cols, group, std=None):
    """Codes over all 16 values, scales and biases of both signs of a matrix of about `std`."""
    std = std or cols**-0.5
    codes = torch.randint(-(2**31), 2**31, (*lead, rows, cols // 8), dtype=torch.int32, device="cuda", generator=gen)
    shape = (*lead, rows, cols // group)
    scales = std / 4.6 * (0.5 + torch.rand(shape, device="cuda", generator=gen))
    biases = -7.5 * scales * (1 + 0.2 * torch.randn(shape, device="cuda", generator=gen))
    sign = torch.where(torch.rand(shape, device="cuda", generator=gen) < 0.1, -1.0, 1.0)
    return codes, (sign * scales).half(), (sign * biases).half()


def floats64(p):
    """(weights, magnitudes |code scale| + |bias|) in float64."""
    codes, scales, biases = p
    q = torch.stack([(codes >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2).double()
    each = q.shape[-1] // scales.shape[-1]
    s, b = (t.double().repeat_interleave(each, -1) for t in (scales, biases))
    return q * s + b, q * s.abs() + b.abs()


def gen_of(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def sums(cols, group):
    return (4 * cols / 32 + 3 * cols / group + 40) * 2.0**-23


def last(y, dtype):
    return y.abs() * torch.finfo(dtype).eps / 2 + (2.0**-25 if dtype == F16 else 0)


def product64(x, p, group, dtype=None):
    """x W^T in float64 and how far a kernel's may be from it."""
    w, m = floats64(p)
    y = x.double() @ w.mT
    off = sums(w.shape[-1], group) * (x.double().abs() @ m.mT)
    return (y, off if dtype is None else off + last(y, dtype))


def glu64(x, gate, up, group, dtype, share=None, rounded=False, apart=False):
    """silu(gate x) up x (times share) in float64, and its tolerance once rounded to dtype (a block keeps more of it);
    rounded: of products whose weights are rounded to float16; apart: that are rounded to float16 themselves."""
    (g, eg), (u, eu) = product64(x, gate, group), product64(x, up, group)
    if rounded:
        eg, eu = (e + x.double().abs() @ last(floats64(p)[0], F16).mT for e, p in ((eg, gate), (eu, up)))
    if apart:
        eg, eu = eg + last(g, F16), eu + last(u, F16)
    a = g * torch.sigmoid(g)
    h, off = a * u, 1.1 * eg * u.abs() + a.abs() * eu + 1.1 * eg * eu
    off = off + (a * u).abs() * 2.0**-20  # float32 exp, quotient and products
    if share is not None:
        h, off = h * share, off * share.abs()
    return h, off + last(h, dtype)


def close(got, want, off):
    assert got.shape == want.shape
    d = (got.double() - want).abs()
    bad = d > off
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((d / off).max()):.2f} of the tolerance"


# ---- floats to codes and back


def quantize_plain(w, group):
    g = w.float().cpu().reshape(*w.shape[:-1], -1, group)
    lo, hi = g.amin(-1), g.amax(-1)
    s, b = ((hi - lo) / torch.full_like(hi, 15)).half(), lo.half()
    sf, bf = s.float()[..., None], b.float()[..., None]
    q = torch.where(sf > 0, ((g - bf) / sf).round().clamp(0, 15), torch.zeros_like(g))
    q = q.reshape(*w.shape[:-1], -1, 8).to(torch.int64)
    words = sum(q[..., i] << (4 * i) for i in range(8))
    return (words - ((words >> 31) << 32)).to(torch.int32), s, b


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lead, blocks", [((1,), 1), ((7,), 3), ((3, 5), 2), ((257,), 9)])
def test_codes_scales_and_biases_are_the_formulas(cuda, group, dtype, lead, blocks):
    w = (0.02 * torch.randn(*lead, blocks * group, device=cuda, generator=gen_of(1))).to(dtype)
    w[..., :group] = 0.25  # a constant group
    if blocks > 1:
        w[..., group : 2 * group] = torch.arange(group, device=cuda).to(dtype) / 16  # many values on a border of two codes
    got = affine.quantize(w, group)
    for g, p in zip(got, quantize_plain(w, group)):
        assert g.dtype == p.dtype and torch.equal(g.cpu(), p)
    for out in (F16, F32):
        back = affine.dequantize(*got, group, dtype=out)
        q = torch.stack([(got[0] >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2).float()
        want = (q * got[1].float().repeat_interleave(group, -1) + got[2].float().repeat_interleave(group, -1)).to(out)
        assert back.shape == w.shape and torch.equal(back, want)


def test_a_float_is_within_its_groups_step(cuda):
    # half a step, and the roundings of scale (15 steps of it at most) and bias to float16
    w = 0.02 * torch.randn(64, 512, device=cuda, generator=gen_of(2))
    codes, s, b = affine.quantize(w, 64)
    back = affine.dequantize(codes, s, b, 64, dtype=F32)
    step = s.float().repeat_interleave(64, -1)
    slack = step * (0.5 + 15 * 2.0**-11) + b.float().abs().repeat_interleave(64, -1) * 2.0**-11 + 1e-7
    assert ((back - w).abs() <= slack).all()


def test_groups_that_are_not_finite_stay_alone(cuda):
    w = torch.randn(4, 256, device=cuda, generator=gen_of(3))
    w[0, 5], w[1, 70], w[2, 130] = float("nan"), float("inf"), 1e30
    codes, s, b = affine.quantize(w, 64)
    back = affine.dequantize(codes, s, b, 64, dtype=F32)
    bad = ~torch.isfinite(back).reshape(4, 4, 64).all(-1)
    assert bad.nonzero().tolist() == [[0, 0], [1, 1], [2, 2]]


def test_conversions_take_views_and_empty_tensors(cuda):
    w = torch.randn(40, 300, device=cuda, generator=gen_of(4)).half()
    part = w[3::2, 7:263]
    for a, b in zip(affine.quantize(part, 64), affine.quantize(part.clone(), 64)):
        assert torch.equal(a, b)
    codes, s, b = affine.quantize(w[:0, :128], 64)
    assert codes.shape == (0, 16) and affine.dequantize(codes, s, b).shape == (0, 128)


@pytest.mark.parametrize("experts, rows, cols, group", [(1, 1, 32, 32), (3, 17, 160, 32), (2, 40, 320, 64), (1, 33, 384, 128)])
def test_the_layout_gives_the_floats_back(cuda, experts, rows, cols, group):
    p = parts(gen_of(5), (experts,), rows, cols, group)
    stack = affine.QuantizedSwitchLinear(*p, group_size=group)
    for dtype in (F16, F32):
        assert torch.equal(stack.floats(dtype), affine.dequantize(*p, group, dtype=dtype))


# ---- one layer

SHAPES = [(1, 32, 32), (15, 96, 32), (16, 64, 64), (17, 128, 128), (100, 1056, 32), (640, 2560, 64), (33, 4736, 64),
          (2051, 384, 128), (48, 8192, 128)]


@pytest.mark.parametrize("rows, cols, group", SHAPES)
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16, 17, 33, 40, 133, 500])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_layer_is_its_definition(cuda, rows, cols, group, tokens, dtype):
    gen = gen_of(tokens + rows)
    p = parts(gen, (), rows, cols, group)
    x = torch.randn(tokens, cols, device=cuda, generator=gen).to(dtype)
    got = affine.QuantizedLinear(*p, group_size=group)(x)
    assert got.dtype == dtype
    close(got, *layer64(x, p, group, dtype))


def layer64(x, p, group, dtype, rounded=False):
    """More than 16 float16 tokens may multiply weights rounded to float16: half a step of each, or of a subnormal."""
    y, off = product64(x, p, group, dtype)
    if dtype == F16 and (rounded or x.shape[0] > 16):
        off = off + x.double().abs() @ last(floats64(p)[0], F16).mT
    return y, off


@pytest.mark.parametrize("rows, cols, group", [(640, 2560, 64), (1000, 1056, 32), (5000, 160, 32), (2051, 384, 128),
                                               (9000, 128, 64), (4096, 4128, 32)])
@pytest.mark.parametrize("tokens", [129, 700, 1500, 2311])
def test_a_prompt_is_its_definition(cuda, rows, cols, group, tokens):
    gen = gen_of(tokens)
    p = parts(gen, (), rows, cols, group)
    x = torch.randn(tokens, cols, device=cuda, generator=gen).half()
    layer = affine.QuantizedLinear(*p, group_size=group)
    for _ in range(3):
        close(layer(x), *layer64(x, p, group, F16))
    assert not affine.failed()


@pytest.mark.parametrize("scale", [2.0**-13, 300.0])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_layer_takes_small_and_large_activations(cuda, scale, dtype):
    # float16 subnormals among the small ones: the products are exact all the same
    gen = gen_of(9)
    p = parts(gen, (), 48, 512, 64)
    x = (scale * torch.randn(3, 512, device=cuda, generator=gen)).to(dtype)
    close(affine.QuantizedLinear(*p, group_size=64)(x), *product64(x, p, 64, dtype))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_token_has_the_same_bits_alone_and_in_a_window(cuda, dtype):
    gen = gen_of(11)
    for rows, cols, group in ((640, 2560, 64), (4100, 1056, 32)):
        layer = affine.QuantizedLinear(*parts(gen, (), rows, cols, group), group_size=group)
        x = torch.randn(16, cols, device=cuda, generator=gen).to(dtype)
        whole = layer(x)
        assert torch.equal(whole, torch.cat([layer(x[i : i + 1]) for i in range(16)]))
        assert torch.equal(whole[:5], layer(x[:5]))


def test_a_layer_takes_views_leads_and_no_tokens(cuda):
    gen = gen_of(12)
    layer = affine.QuantizedLinear(*parts(gen, (), 96, 256, 64), group_size=64)
    x = torch.randn(6, 9, 300, device=cuda, generator=gen).half()
    view = x.transpose(0, 1)[::2, :, 3:259]
    assert torch.equal(layer(view), layer(view.contiguous()))
    flat = torch.randn(1 + 2 * 256, device=cuda, generator=gen).half()
    off = flat[1:].view(2, 256)  # contiguous, off a 16-byte boundary
    assert off.data_ptr() % 16 and torch.equal(layer(off), layer(off.clone()))
    assert layer(x[:0, :, :256]).shape == (0, 9, 96)
    assert layer(x[0, 0, :256]).shape == (96,)


@pytest.mark.parametrize("rows, cols, tokens, dtype", [(16, 2**21, 2, F16), (3, 2**21, 1, F32), (40, 2**20, 20, F16), (200000, 32, 1, F16),
                                                       (200000, 32, 40, F16)])
def test_long_rows_and_many_rows(cuda, rows, cols, tokens, dtype):
    gen = gen_of(18)
    p = parts(gen, (), rows, cols, 32)
    x = torch.randn(tokens, cols, device=cuda, generator=gen).to(dtype)
    want, off = product64(x, p, 32, dtype)
    if tokens > 16:  # (weights rounded to float16)
        off = off + x.double().abs() @ (floats64(p)[0].abs().mT * 2.0**-11 + 2.0**-25)
    close(affine.QuantizedLinear(*p, group_size=32)(x), want, off)


def test_a_copy_of_a_layer_has_weights_of_its_own(cuda):
    gen = gen_of(19)
    layer = affine.QuantizedLinear(*parts(gen, (), 48, 128, 64))
    x = torch.randn(3, 128, device=cuda, generator=gen).half()
    want = layer(x)
    other = copy.deepcopy(layer)
    layer.packed.zero_()
    torch.cuda.synchronize()  # (a layer's weights are not to be written by the launch before its product)
    assert torch.equal(other(x), want) and not layer(x).any()


def test_one_row_of_floats(cuda):
    w = torch.randn(128, device=cuda, generator=gen_of(21))
    p = affine.quantize(w, 32)
    assert [t.shape for t in p] == [(16,), (4,), (4,)]
    assert torch.equal(affine.dequantize(*p, 32), affine.dequantize(*affine.quantize(w[None], 32), 32)[0])


def test_what_is_not_finite_stays_in_its_token(cuda):
    gen = gen_of(13)
    layer = affine.QuantizedLinear(*parts(gen, (), 64, 256, 64), group_size=64)
    x = torch.randn(5, 256, device=cuda, generator=gen).half()
    want = layer(x)
    for bad in (float("inf"), float("nan")):
        y = x.clone()
        y[2, 77] = bad
        got = layer(y)
        assert not torch.isfinite(got[2]).any() and torch.equal(got[[0, 1, 3, 4]], want[[0, 1, 3, 4]])


# ---- pairs


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens, k, experts", [(1, 1, 1), (1, 4, 9), (5, 3, 4), (40, 2, 3), (30, 32, 40), (700, 3, 7)])
def test_pair_products_are_their_definition(cuda, dtype, tokens, k, experts):
    gen = gen_of(tokens)
    rows, cols, group = 40, 160, 32
    p = parts(gen, (experts,), rows, cols, group)
    stack = affine.QuantizedSwitchLinear(*p, group_size=group)
    idx = torch.randint(0, experts, (tokens, k), device=cuda, generator=gen)  # an expert may come twice in a token
    x = torch.randn(tokens, 1, 1, cols, device=cuda, generator=gen).to(dtype)
    got = stack(x, idx)
    assert got.shape == (tokens, k, 1, rows)
    for e in range(experts):
        t, j = (idx == e).nonzero(as_tuple=True)
        one = [a[e] for a in p]
        want, off = product64(x[t, 0, 0], one, group, dtype)
        if dtype == F16 and tokens * k > affine.MAX_PAIRS:  # (by tiles: half a step of each weight, rounded to float16)
            off = off + x[t, 0, 0].double().abs() @ last(floats64(one)[0], F16).mT
        close(got[t, j, 0], want, off)
    each = stack(x.expand(tokens, k, 1, cols), idx)  # a row of its own for every pair
    close(each.double(), got.double(), last(got.double(), dtype) * 2 + sums(cols, group) * 8)


def test_pairs_of_no_expert_are_left_as_they_were(cuda):
    gen = gen_of(20)
    stack = affine.QuantizedSwitchLinear(*parts(gen, (6,), 33, 64, 64), group_size=64)
    x = torch.randn(4, 64, device=cuda, generator=gen).half()
    idx = torch.tensor([[0, 6], [5, 5], [7, -1], [2, 1]], dtype=torch.int32, device=cuda)
    out = torch.full((8, 33), 7.0, dtype=F16, device=cuda)
    spec = _lib.SmoeQ4Product(dtype=1, group=64, x=x.data_ptr(), cols=64, stack=stack.data_ptr, rows=33, experts=6,
                              idx=idx.data_ptr(), pairs=8, share=2, out=out.data_ptr())
    _lib.call("smoe_q4_product", ctypes.byref(spec), _lib.stream())
    want = stack(x[:, None, None], idx.clamp(0, 5))[:, :, 0].reshape(8, 33)
    out_of = torch.tensor([0, 1, 0, 0, 1, 1, 0, 0], dtype=torch.bool, device=cuda)
    assert (out[out_of] == 7).all() and torch.equal(out[~out_of], want[~out_of])


@pytest.fixture
def by_tiles(monkeypatch):
    """Every float16 call of pairs by the tiles of a prompt."""
    monkeypatch.setattr(affine, "_by_tiles", lambda lin, dtype, pairs: dtype == F16 and pairs > 0)


TILES = [(1, 1, 1, 40, 32, 32), (5, 3, 4, 16, 128, 64), (40, 2, 3, 129, 160, 32), (30, 32, 40, 250, 384, 128), (700, 3, 7, 600, 96, 32),
         (2000, 1, 2, 24, 2176, 64), (300, 8, 1024, 33, 64, 64), (1180, 8, 256, 130, 128, 64), (9000, 2, 3, 16, 32, 32)]


@pytest.mark.parametrize("tokens, k, experts, rows, cols, group", TILES)
def test_pair_products_by_tiles_are_their_definition(cuda, by_tiles, tokens, k, experts, rows, cols, group):
    gen = gen_of(tokens + rows)
    p = parts(gen, (experts,), rows, cols, group)
    stack = affine.QuantizedSwitchLinear(*p, group_size=group)
    idx = torch.randint(0, experts, (tokens, k), dtype=torch.int32, device=cuda, generator=gen)
    x = torch.randn(tokens, 1, 1, cols, device=cuda, generator=gen).half()
    got = stack(x, idx)
    assert got.shape == (tokens, k, 1, rows)
    for e in range(experts):
        t, j = (idx == e).nonzero(as_tuple=True)
        if len(t):
            close(got[t, j, 0], *layer64(x[t, 0, 0], [a[e] for a in p], group, F16, rounded=True))
    assert torch.equal(stack(x.expand(tokens, k, 1, cols), idx), got) and torch.equal(stack(x, idx), got)
    assert not affine.failed()


@pytest.mark.parametrize("tokens, k, experts, hidden, ffn, group, down_group", [(9, 2, 3, 96, 64, 32, 64), (200, 6, 17, 320, 160, 32, 32),
                                                                               (700, 4, 5, 256, 384, 128, 64)])
def test_experts_by_tiles_are_their_definition(cuda, by_tiles, tokens, k, experts, hidden, ffn, group, down_group):
    gen = gen_of(tokens)
    r, _, glu, _ = make_experts(gen, experts, hidden, ffn, 128, group, down_group)
    x = torch.randn(tokens, hidden, device=cuda, generator=gen).half()
    idx = torch.rand(tokens, experts, device=cuda, generator=gen).argsort(-1)[:, :k] if k <= experts else torch.randint(
        0, experts, (tokens, k), device=cuda, generator=gen)
    idx[3, 1], idx[5] = experts, -1  # pairs of no expert
    y = glu(x, idx)
    for e in range(experts):
        t, j = (idx == e).nonzero(as_tuple=True)
        gate, up, down = ([a[e] for a in p] for p in r)
        h, eh = glu64(x[t], gate, up, group, F16, rounded=True)
        want, off = layer64(h, down, down_group, F16, rounded=True)
        close(y[t, j], want, off + eh @ floats64(down)[0].abs().mT * 1.01)


def test_pairs_of_no_expert_by_tiles_are_left_as_they_were(cuda):
    gen = gen_of(24)
    stack = affine.QuantizedSwitchLinear(*parts(gen, (6,), 33, 64, 64), group_size=64)
    x = torch.randn(4, 64, device=cuda, generator=gen).half()
    idx = torch.tensor([[0, 6], [5, 5], [7, -1], [2, 1]], dtype=torch.int32, device=cuda)
    want = stack(x[:, None, None], idx.clamp(0, 5))[:, :, 0].reshape(8, 33)
    tiles = affine._Tiles(stack, idx.reshape(-1), 2)
    a = x.index_select(0, tiles.row)
    for dtype in (F16, F32):
        out = tiles.product(stack, a, torch.full((8, 33), 7.0, dtype=dtype, device=cuda), True)
        out_of = torch.tensor([0, 1, 0, 0, 1, 1, 0, 0], dtype=torch.bool, device=cuda)
        assert (out[out_of] == 7).all() and (out[~out_of] - want[~out_of].to(dtype)).abs().max() < 0.02
        none = affine._Tiles(stack, torch.full((8,), 9, dtype=torch.int32, device=cuda), 2)
        assert (none.product(stack, a[: none.count * 16], torch.full((8, 33), 7.0, dtype=dtype, device=cuda), True) == 7).all()


def test_what_is_not_finite_stays_in_its_pairs_by_tiles(cuda, by_tiles):
    gen = gen_of(25)
    _, _, glu, _ = make_experts(gen, 5, 160, 96, 64, 32)
    x = torch.randn(40, 160, device=cuda, generator=gen).half()
    idx = torch.randint(0, 5, (40, 3), dtype=torch.int32, device=cuda, generator=gen)
    want = glu(x, idx)
    x[0, 5], x[17, 159] = float("nan"), float("inf")  # (token 0's row stands in the slots without a pair, too)
    got = glu(x, idx)
    hit = torch.zeros(40, dtype=torch.bool, device=cuda)
    hit[[0, 17]] = True
    assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], want[~hit])


def test_no_pairs(cuda):
    gen = gen_of(22)
    _, _, glu, _ = make_experts(gen, 4, 128, 64, 64, 64)
    x = torch.randn(3, 128, device=cuda, generator=gen).half()
    none = torch.zeros(3, 0, dtype=torch.int32, device=cuda)
    assert glu(x, none).shape == (3, 0, 128) and glu(x[:0], none[:0]).shape == (0, 0, 128)
    assert glu(x[:0], torch.zeros(0, 2, dtype=torch.int32, device=cuda)).shape == (0, 2, 128)
    assert glu.gate_proj(x[:, None, None], none).shape == (3, 0, 1, 64)


# ---- the experts and the block


def make_experts(gen, experts, hidden, ffn, shared, group, down_group=None):
    down_group = down_group or group
    r = [parts(gen, (experts,), ffn, hidden, group), parts(gen, (experts,), ffn, hidden, group),
         parts(gen, (experts,), hidden, ffn, down_group)]
    s = [parts(gen, (), shared, hidden, group), parts(gen, (), shared, hidden, group),
         parts(gen, (), hidden, shared, down_group)]
    gs = (group, group, down_group)
    glu = affine.QuantizedSwitchGLU(*(affine.QuantizedSwitchLinear(*p, group_size=g) for p, g in zip(r, gs)))
    mlp = affine.QuantizedMLP(*(affine.QuantizedLinear(*p, group_size=g) for p, g in zip(s, gs)))
    return r, s, glu, mlp


def moe64(x, r, s, idx, w, g, group, down_group, dtype, rounded=False):
    """The block behind its route in float64 and its tolerance; idx past the experts adds nothing. Past 64 tokens the
    experts' outputs, the shared expert's, its gate (and their product) and the sum of the experts' are rounded to dtype
    each: three half steps of every term at most (in float32 the sum's k additions and products besides). rounded: float16
    weights, and the shared expert's gate and up, too."""
    tokens, hidden = x.shape
    out, off = torch.zeros(tokens, hidden, dtype=torch.float64, device=x.device), torch.zeros(tokens, hidden, dtype=torch.float64, device=x.device)

    def add(t, mats, share, members):
        h, eh = glu64(x[t], mats[0], mats[1], group, dtype, share[:, None], rounded, rounded)
        wd, md = floats64(mats[2])
        n = sums(wd.shape[-1] * members, down_group)  # (one sum over every expert's columns)
        out.index_add_(0, t, h @ wd.mT)
        off.index_add_(0, t, eh @ wd.abs().mT + n * ((h.abs() + eh) @ md.mT))
        if rounded:
            off.index_add_(0, t, (h.abs() + eh) @ last(wd, F16).mT)
        if tokens > 64:
            y = h @ wd.mT
            each = y.abs() * torch.finfo(dtype).eps / 2 + (2.0**-25 if dtype == F16 else 0)
            off.index_add_(0, t, 1.01 * each * (3 if dtype == F16 else 2 * members + 3))

    members = idx.shape[1] + 1
    for e in range(r[0][0].shape[0]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if len(t):
            add(t, [[a[e] for a in p] for p in r], w[t, j].double(), members)
    gate = torch.sigmoid(g.double().reshape(-1))
    add(torch.arange(tokens, device=x.device), s, gate, members)
    return out, off + last(out, dtype)


MOE = [(1, 9, 3, 96, 32, 64, 32, 32), (2, 4, 4, 128, 64, 192, 64, 64), (5, 24, 4, 1056, 352, 544, 32, 32),
       (8, 40, 8, 256, 128, 128, 128, 64), (9, 7, 2, 192, 320, 64, 64, 32), (17, 33, 10, 128, 64, 64, 32, 64),
       (33, 5, 1, 64, 32, 32, 32, 32), (64, 64, 8, 256, 192, 320, 64, 64), (70, 12, 3, 64, 64, 64, 64, 64),
       (3, 300, 10, 2560, 640, 640, 64, 64)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens, experts, k, hidden, ffn, shared, group, down_group", MOE)
def test_a_block_behind_its_route_is_its_definition(cuda, dtype, tokens, experts, k, hidden, ffn, shared, group, down_group):
    gen = gen_of(tokens + hidden)
    r, s, glu, mlp = make_experts(gen, experts, hidden, ffn, shared, group, down_group)
    x = torch.randn(tokens, hidden, device=cuda, generator=gen).to(dtype)
    idx = torch.rand(tokens, experts, device=cuda, generator=gen).argsort(-1)[:, :k].to(torch.int32)
    w = torch.softmax(torch.randn(tokens, k, device=cuda, generator=gen), -1)
    g = torch.randn(tokens, 1, device=cuda, generator=gen).to(dtype)
    got = affine.moe(glu, mlp, x, idx, w, g)
    close(got, *moe64(x, r, s, idx, w, g, group, down_group, dtype))
    # choices of no expert, the same expert twice, tokens without any expert
    idx[::2, 0] = experts
    if k > 1:
        idx[:, 1] = idx[:, -1]
    idx[-1] = -1
    close(affine.moe(glu, mlp, x, idx, w, g), *moe64(x, r, s, idx, w, g, group, down_group, dtype))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens, shared", [(3, 0), (3, 96), (64, 0)])
def test_a_block_without_a_shared_expert_or_its_gate(cuda, dtype, tokens, shared):
    gen = gen_of(33)
    hidden, ffn, experts, k, group = 160, 96, 2048, 32, 32
    r, s, glu, mlp = make_experts(gen, experts, hidden, ffn, shared or 32, group)
    x = torch.randn(tokens, hidden, device=cuda, generator=gen).to(dtype)
    idx = torch.randint(0, experts, (tokens, k), dtype=torch.int32, device=cuda, generator=gen)
    w = torch.rand(tokens, k, device=cuda, generator=gen)
    out = torch.full((tokens, hidden), 7.0, dtype=dtype, device=cuda)
    spec = _lib.SmoeQ4Moe(dtype=_lib.dtype_code(dtype), group=group, down_group=group, tokens=tokens, hidden=hidden,
                          experts=experts, k=k, ffn=ffn, shared_ffn=shared, x=x.data_ptr(), idx=idx.data_ptr(),
                          weights=w.data_ptr(), gate=glu.gate_proj.data_ptr, up=glu.up_proj.data_ptr,
                          down=glu.down_proj.data_ptr, out=out.data_ptr())
    if shared:
        spec.sgate, spec.sup, spec.sdown = (p.data_ptr for p in (mlp.gate_proj, mlp.up_proj, mlp.down_proj))
    nbytes = int(_lib.lib().smoe_q4_moe_workspace_size(tokens, k, hidden, ffn, shared))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
    _lib.call("smoe_q4_moe", ctypes.byref(spec), _lib.ptr(ws), nbytes, _lib.stream())
    # (the gate of a shared expert that has none is 1; one that is not there has weights of zero)
    want = moe64(x, r, s if shared else [[t * 0 for t in p] for p in s], idx, w, torch.full((tokens, 1), 40.0, device=cuda), group,
                 group, dtype)
    close(out, *want)


def test_a_router_at_any_address(cuda):
    gen = gen_of(35)
    _, _, block, router, sgate = make_block(gen, 20, 256, 128, 192, 64, 4)
    x = torch.randn(5, 256, device=cuda, generator=gen).half()
    want = block(x)

    def moved(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape).copy_(t)

    other = fused.SparseMoeBlock(moved(router), block.switch_mlp, block.shared_expert, moved(sgate), 4)
    assert torch.equal(other(moved(x)), want)
    assert torch.equal(other(torch.stack((x, x), -1)[..., 1]), want)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_the_experts_alone_are_their_definition(cuda, dtype):
    gen = gen_of(31)
    r, s, glu, mlp = make_experts(gen, 6, 192, 96, 160, 32)
    x = torch.randn(11, 192, device=cuda, generator=gen).to(dtype)
    idx = torch.randint(0, 6, (11, 3), device=cuda, generator=gen)
    y = glu(x, idx)
    for e in range(6):
        t, j = (idx == e).nonzero(as_tuple=True)
        gate, up, down = ([a[e] for a in p] for p in r)
        h, eh = glu64(x[t], gate, up, 32, dtype)
        wd, md = floats64(down)
        want = h @ wd.mT
        close(y[t, j], want, eh @ wd.abs().mT + sums(96, 32) * ((h.abs() + eh) @ md.mT) + last(want, dtype))
    h, eh = glu64(x, s[0], s[1], 32, dtype)
    wd, md = floats64(s[2])
    want = h @ wd.mT
    close(mlp(x), want, eh @ wd.abs().mT + sums(160, 32) * ((h.abs() + eh) @ md.mT) + last(want, dtype))


@pytest.mark.parametrize("tokens, experts, hidden, k", [(1, 512, 2560, 10), (1, 1, 32, 1), (2, 33, 1056, 4), (8, 256, 4096, 8),
                                                        (9, 15, 96, 15), (17, 300, 2048, 32), (33, 2048, 64, 3), (64, 511, 512, 10)])
def test_the_route_of_a_window_is_its_definition(cuda, tokens, experts, hidden, k):
    gen = gen_of(tokens + experts)
    router = (hidden**-0.5 * torch.randn(experts, hidden, device=cuda, generator=gen)).half()
    sgate = (hidden**-0.5 * torch.randn(1, hidden, device=cuda, generator=gen)).half()
    x = torch.randn(tokens, hidden, device=cuda, generator=gen).half()
    gate, shared = fused.WindowLinear(router), fused.WindowLinear(sgate)
    # one addition for every column in the order of any sum, at most 2^-23 of the magnitudes each
    logits, off = x.double() @ router.double().mT, hidden * 2.0**-23 * (x.double().abs() @ router.double().abs().mT)
    for _ in range(3):  # (the counter is left as it was found)
        idx, w, g = fused.route_window(gate, shared, x, k)
        idx = idx.view(torch.int32).long()
        chosen = logits.gather(1, idx)
        slack = off.max()
        assert (idx.sort(-1).values.diff(dim=-1) > 0).all() and (chosen.diff(dim=-1) <= 2 * slack).all()
        left = logits.scatter(1, idx, -torch.inf).amax(-1)
        assert (chosen.amin(-1) >= left - 2 * slack).all()
        close(w, torch.softmax(chosen, -1), (2 * slack + 2.0**-20) * torch.softmax(chosen, -1) + 1e-30)
        want = x.double() @ sgate.double().mT
        close(g, want, hidden * 2.0**-23 * (x.double().abs() @ sgate.double().abs().mT) + last(want, F16))
    assert fused.route_window(gate, shared, x.float(), k) is None
    assert fused.route_window(gate, shared, x.expand(65, -1, -1).reshape(-1, hidden), k) is None


def test_equal_logits_go_to_the_lower_index(cuda):
    router = torch.ones(40, 64, dtype=F16, device=cuda)
    router[7] = 0.5
    x = torch.ones(3, 64, dtype=F16, device=cuda)
    idx, w, _ = fused.route_window(fused.WindowLinear(router), fused.WindowLinear(router[:1]), x, 9)
    assert idx.view(torch.int32).tolist() == [[0, 1, 2, 3, 4, 5, 6, 8, 9]] * 3
    assert (w - 1 / 9).abs().max() < 2.0**-20


def make_block(gen, experts, hidden, ffn, shared, group, k, from_floats=False):
    router = (hidden**-0.5 * torch.randn(experts, hidden, device="cuda", generator=gen)).half()
    sgate = (hidden**-0.5 * torch.randn(1, hidden, device="cuda", generator=gen)).half()
    if not from_floats:
        r, s, glu, mlp = make_experts(gen, experts, hidden, ffn, shared, group)
    else:
        def floats(*shape):
            return (shape[-1] ** -0.5 * torch.randn(*shape, device="cuda", generator=gen)).half()

        r = [affine.quantize(floats(experts, *d), group) for d in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
        s = [affine.quantize(floats(*d), group) for d in ((shared, hidden), (shared, hidden), (hidden, shared))]
        glu = affine.QuantizedSwitchGLU(*(affine.QuantizedSwitchLinear(*p, group_size=group) for p in r))
        mlp = affine.QuantizedMLP(*(affine.QuantizedLinear(*p, group_size=group) for p in s))
    return r, s, fused.SparseMoeBlock(router, glu, mlp, sgate, k), router, sgate


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens", [1, 6, 64, 90])
def test_floats_made_4_bit_and_run_as_a_block(cuda, dtype, tokens):
    gen = gen_of(41)
    r, s, block, router, sgate = make_block(gen, 20, 256, 128, 192, 64, 4, from_floats=True)
    x = torch.randn(tokens, 256, device=cuda, generator=gen).to(dtype)
    got = block(x)
    idx, w = fused.top_k_softmax(block.gate(x), 4)
    logits = x.double() @ router.double().mT
    idx = idx.view(torch.int32)
    assert torch.equal(idx.long().sort(-1).values, logits.topk(4, -1).indices.sort(-1).values)
    g = block.shared_expert_gate(x).to(dtype)
    close(got, *moe64(x, r, s, idx, w, g, 64, 64, dtype))


def test_a_graph_replays_the_eager_bits(cuda):
    gen = gen_of(43)
    _, _, block, _, _ = make_block(gen, 40, 256, 128, 192, 64, 5)
    for tokens in (1, 5, 20, 500):
        xs = [torch.randn(tokens, 256, device=cuda, generator=gen).half() for _ in range(3)]
        eager = [block(x).clone() for x in xs]
        step = fused.GraphedBlock(block, tokens, 256, F16, cuda)
        for _ in range(2):
            for x, want in zip(xs, eager):
                assert torch.equal(step(x), want)
    assert not affine.failed()


@pytest.mark.parametrize("tokens, experts, k, hidden, ffn, shared, group", [(700, 20, 4, 256, 192, 1120, 32), (260, 12, 10, 1024, 64, 2048, 64)])
def test_a_prompt_through_the_experts_and_their_combine(cuda, tokens, experts, k, hidden, ffn, shared, group):
    gen = gen_of(tokens)
    r, s, glu, mlp = make_experts(gen, experts, hidden, ffn, shared, group)
    assert tokens * k > affine.MAX_PAIRS and mlp._apart(tokens) == (tokens == 700)
    x = torch.randn(tokens, hidden, device=cuda, generator=gen).half()
    idx = torch.rand(tokens, experts, device=cuda, generator=gen).argsort(-1)[:, :k].to(torch.int32)
    w = torch.softmax(torch.randn(tokens, k, device=cuda, generator=gen), -1)
    g = torch.randn(tokens, 1, device=cuda, generator=gen).half()
    idx[::7, 0], idx[11] = experts, -1  # choices of no expert
    close(affine.moe(glu, mlp, x, idx, w, g), *moe64(x, r, s, idx, w, g, group, group, F16, rounded=True))
    assert not affine.failed()


def test_a_prompt_in_several_parts(cuda, monkeypatch):
    gen = gen_of(46)
    _, _, block, _, _ = make_block(gen, 40, 256, 128, 192, 64, 5)
    x = torch.randn(900, 256, device=cuda, generator=gen).half()
    idx = torch.randint(0, 40, (900, 5), dtype=torch.int32, device=cuda, generator=gen)
    up = block.switch_mlp.up_proj
    want = block(x), up(x[:, None, None], idx)
    monkeypatch.setattr(affine, "TILE_PAIRS", 1111)
    assert torch.equal(block(x), want[0]) and torch.equal(up(x[:, None, None], idx), want[1])
    # (a part's calls are those of a prompt of its length, whose kernels may be others)
    w, g = torch.rand(900, 5, device=cuda, generator=gen), torch.randn(900, 1, device=cuda, generator=gen).half()

    def moe(a, b):
        return affine.moe(block.switch_mlp, block.shared_expert, x[a:b], idx[a:b], w[a:b], g[a:b])

    parts_of = torch.cat((moe(0, 500), moe(500, 900)))
    monkeypatch.setattr(affine, "COMBINE_TOKENS", 500)
    assert torch.equal(moe(0, 900), parts_of)


def test_two_graphs_and_an_eager_call_at_once(cuda):
    gen = gen_of(44)
    _, _, block, _, _ = make_block(gen, 40, 256, 128, 192, 64, 5)
    xs = [torch.randn(4, 256, device=cuda, generator=gen).half() for _ in range(3)]
    want = [block(x).clone() for x in xs]
    steps = [fused.GraphedBlock(block, 4, 256, F16, cuda) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(50):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(steps[i](xs[i]) if i < 2 else block(xs[i]))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def test_calls_that_are_refused(cuda):
    gen = gen_of(45)
    p = parts(gen, (), 32, 128, 64)
    layer = affine.QuantizedLinear(*p, group_size=64)
    x = torch.zeros(2, 128, dtype=F16, device=cuda)
    for bad, match in ((x.bfloat16(), "not supported"), (x[:, :64], "do not end"), (x.cpu(), "CUDA"), (x.long(), "not supported")):
        with pytest.raises(ValueError, match=match):
            layer(bad)
    with pytest.raises(ValueError, match="float16"):
        affine.QuantizedLinear(p[0], p[1].float(), p[2])
    with pytest.raises(ValueError, match="no matrix"):
        affine.QuantizedLinear(*p, group_size=32)
    with pytest.raises(ValueError, match="32-bit"):
        affine.QuantizedLinear(p[0].long(), p[1], p[2])
    with pytest.raises(ValueError, match="without weights"):
        affine.QuantizedLinear(*(t[:0] for t in p))
    with pytest.raises(ValueError, match="whole number"):
        affine.quantize(torch.zeros(3, 100, device=cuda))
    with pytest.raises(ValueError, match="not supported"):
        affine.quantize(torch.zeros(3, 64, device=cuda).bfloat16())
    r, s, glu, mlp = make_experts(gen, 4, 128, 64, 64, 64)
    with pytest.raises(ValueError, match="one shape"):
        affine.QuantizedMLP(layer, affine.QuantizedLinear(*parts(gen, (), 16, 128, 64)), layer)
    with pytest.raises(ValueError, match="down must"):
        affine.QuantizedSwitchGLU(glu.gate_proj, glu.up_proj, glu.gate_proj)
    idx = torch.zeros(2, 2, dtype=torch.int32, device=cuda)
    w, g = torch.zeros(2, 2, device=cuda), torch.zeros(2, 1, dtype=F16, device=cuda)
    for args in ((x, idx[:1], w, g), (x, idx, w.half(), g), (x, idx, w, g.float()), (x, idx, w, g[:1])):
        with pytest.raises(ValueError):
            affine.moe(glu, mlp, *args)
    with pytest.raises(ValueError):
        glu(x, idx[:1])
