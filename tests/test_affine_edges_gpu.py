"""Calls of the 4-bit layers at the edges of what they allow, against their definition in 64 bits. The tolerances are those
derived in test_affine_gpu.py: the worst case of every rounding, which is a large part of the result where its terms cancel.
Weights and activations here are positive, so that nothing cancels and a tolerance is a small fraction of the result."""

import ctypes

import numpy as np
import pytest

from oracle import quants as Q

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from strata_mlx_b200 import _lib, affine, blocks, fused  # noqa: E402
from test_affine_gpu import F16, F32, MOE, SHAPES, close, floats64, gen_of, glu64, last, layer64, moe64, parts, product64  # noqa: E402


def positive(gen, lead, rows, cols, group):
    """Codes over all 16 values, scales and biases of a matrix of weights from 0.005 to 0.05."""
    codes = torch.randint(-(2**31), 2**31, (*lead, rows, cols // 8), dtype=torch.int32, device="cuda", generator=gen)
    shape = (*lead, rows, cols // group)
    scales = 0.001 * (1 + torch.rand(shape, device="cuda", generator=gen))
    biases = 0.005 + 0.01 * torch.rand(shape, device="cuda", generator=gen)
    return codes, scales.half(), biases.half()


def positive_rows(gen, tokens, cols, dtype):
    """Activations that such a matrix takes to about 1.5."""
    return (150 / cols * (0.05 + torch.rand(tokens, cols, device="cuda", generator=gen))).to(dtype)


def positive_experts(gen, experts, hidden, ffn, shared, group, down_group):
    r = [positive(gen, (experts,), *d, n) for *d, n in ((ffn, hidden, group), (ffn, hidden, group), (hidden, ffn, down_group))]
    s = [positive(gen, (), *d, n) for *d, n in ((shared, hidden, group), (shared, hidden, group), (hidden, shared, down_group))]
    gs = (group, group, down_group)
    return (r, s, affine.QuantizedSwitchGLU(*(affine.QuantizedSwitchLinear(*p, group_size=n) for p, n in zip(r, gs))),
            affine.QuantizedMLP(*(affine.QuantizedLinear(*p, group_size=n) for p, n in zip(s, gs))))


def near(got, want, off):
    assert (off <= 0.01 * want).all()
    close(got, want, off)


def block_behind_route(glu, mlp, x, idx, w, g):
    """smoe_q4_moe of one call; mlp None: without a shared expert."""
    gate, down = glu.gate_proj, glu.down_proj
    (tokens, hidden), k, shared = x.shape, idx.shape[1], mlp.gate_proj.output_dims if mlp else 0
    out = torch.full((tokens, hidden), 7.0, dtype=x.dtype, device=x.device)
    spec = _lib.SmoeQ4Moe(dtype=_lib.dtype_code(x.dtype), group=gate.group_size, down_group=down.group_size, tokens=tokens,
                          hidden=hidden, experts=gate.num_experts, k=k, ffn=gate.output_dims, shared_ffn=shared,
                          x=x.data_ptr(), idx=idx.data_ptr(), weights=w.data_ptr(), shared_gate=g.data_ptr(),
                          gate=gate.data_ptr, up=glu.up_proj.data_ptr, down=down.data_ptr, out=out.data_ptr())
    if mlp:
        spec.sgate, spec.sup, spec.sdown = (p.data_ptr for p in (mlp.gate_proj, mlp.up_proj, mlp.down_proj))
    nbytes = int(_lib.lib().smoe_q4_moe_workspace_size(tokens, k, hidden, gate.output_dims, shared))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.call("smoe_q4_moe", ctypes.byref(spec), _lib.ptr(ws), nbytes, _lib.stream())
    return out


# the choices of one token among 12 experts: an expert twice or more, next to and apart from itself, before, between and
# after single ones, beside choices of no expert, more often than a block of rows holds, and all distinct
CHOICES = [[3, 3], [3, 3, 5], [5, 3, 3], [1, 5, 5, 9], [3, 9, 3], [9, 0, 9, 0], [4, 4, 4], [11, 4, 2, 4, 4, 0], [6, -1, 6, 12, 2],
           [7] * 9 + [2], [0] + [7] * 5 + [11], [2, 1, 0] * 10 + [1, 1], [10, 3, 8, 1], [-1, 12]]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hidden, ffn, shared, group, down_group", [(2560, 640, 640, 64, 64), (4096, 1536, 4096, 64, 64),
                                                                    (96, 32, 64, 32, 32), (256, 384, 128, 128, 64)])
def test_one_token_that_names_an_expert_twice(cuda, dtype, hidden, ffn, shared, group, down_group):
    gen = gen_of(hidden + ffn)
    r, s, glu, mlp = positive_experts(gen, 12, hidden, ffn, shared, group, down_group)
    none = [[t * 0 for t in p] for p in s]
    for choice in CHOICES:
        x = positive_rows(gen, 1, hidden, dtype)
        idx = torch.tensor([choice], dtype=torch.int32, device=cuda)
        w = 0.05 + torch.rand(1, len(choice), device=cuda, generator=gen)
        g = torch.randn(1, 1, device=cuda, generator=gen).to(dtype)
        near(affine.moe(glu, mlp, x, idx, w, g), *moe64(x, r, s, idx, w, g, group, down_group, dtype))
        want, off = moe64(x, r, none, idx, w, g, group, down_group, dtype)
        alone = block_behind_route(glu, None, x, idx, w, g)
        if choice == [-1, 12]:
            assert not alone.any()
        else:
            near(alone, want, off)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens, experts, k, hidden, ffn, shared, group, down_group", MOE)
def test_a_block_of_positive_weights(cuda, dtype, tokens, experts, k, hidden, ffn, shared, group, down_group):
    gen = gen_of(tokens + ffn)
    r, s, glu, mlp = positive_experts(gen, experts, hidden, ffn, shared, group, down_group)
    x = positive_rows(gen, tokens, hidden, dtype)
    w = 0.05 + torch.rand(tokens, k, device=cuda, generator=gen)
    g = torch.randn(tokens, 1, device=cuda, generator=gen).to(dtype)
    idx = torch.randint(0, experts, (tokens, k), dtype=torch.int32, device=cuda, generator=gen)  # repeats among them
    near(affine.moe(glu, mlp, x, idx, w, g), *moe64(x, r, s, idx, w, g, group, down_group, dtype))
    idx[::2, 0] = experts
    near(affine.moe(glu, mlp, x, idx, w, g), *moe64(x, r, s, idx, w, g, group, down_group, dtype))


@pytest.mark.parametrize("tokens", [1, 5, 64])
def test_the_shared_gate_is_not_rounded_between_the_route_and_the_block(cuda, tokens):
    # logits of the gate around -9.3, where float16 has steps of 2^-7 and sigmoid follows them in full: a rounded one leaves the
    # result 0.3 % off. The routed experts are zero.
    gen = gen_of(47)
    hidden, ffn, shared, group = 256, 64, 96, 32
    r, s, _, mlp = positive_experts(gen, 6, hidden, ffn, shared, group, group)
    r = [[t * 0 for t in p] for p in r]
    glu = affine.QuantizedSwitchGLU(*(affine.QuantizedSwitchLinear(*p, group_size=group) for p in r))
    router = torch.randn(6, hidden, device=cuda, generator=gen).half()
    sgate = torch.zeros(1, hidden, dtype=F16, device=cuda)
    sgate[0, 0], sgate[0, 1] = -9.3125, -1.0  # a multiple of 2^-7, and what x brings on top of it
    x = 4 * positive_rows(gen, tokens, hidden, F16)
    x[:, 0], x[:, 1] = 1, 2.0**-8 * (0.75 + 0.2 * torch.rand(tokens, device=cuda, generator=gen)).half()
    g = x.double() @ sgate.double().mT
    assert (((g - g.half().double()) / 2.0**-8).abs() > 0.7).all()
    idx, w = torch.zeros(tokens, 2, dtype=torch.int32, device=cuda), torch.zeros(tokens, 2, device=cuda)
    want, off = moe64(x, r, s, idx, w, g, group, group, F16)
    off = off + want * 2.0**-18  # (the gate's sum in float32: a few steps of 2^-24 of 9.3)
    assert (off < 0.002 * want).all()
    got = fused.SparseMoeBlock(router, glu, mlp, sgate, 2)(x)
    assert got.dtype == F16
    close(got, want, off)


@pytest.mark.parametrize("rows, cols, tokens, group", [(1536, 4096, 4096, 64), (4096, 1024, 2048, 128), (9000, 128, 1500, 64),
                                                       (6000, 32, 2311, 32), (128 * 150, 256, 300, 32)])
def test_prompts_with_one_accumulator_or_one_stage_a_job(cuda, rows, cols, tokens, group):
    # several jobs a CTA on one accumulator (more than 160 tokens a job), and jobs that one group of decoders decodes alone
    gen = gen_of(rows + cols)
    p = positive(gen, (), rows, cols, group)
    layer = affine.QuantizedLinear(*p, group_size=group)
    x = positive_rows(gen, tokens, cols, F16)
    want = layer(x)
    near(want, *layer64(x, p, group, F16))
    for _ in range(20):
        assert torch.equal(layer(x), want)
    assert not affine.failed()


@pytest.mark.parametrize("cols, group", [(256, 64), (1024, 32), (512, 128)])
def test_small_terms_beside_large_ones_that_cancel(cuda, cols, group):
    # In every 32 columns a pair of +-32768 with equal codes in each half of the columns of an MMA step: their terms cancel
    # exactly, and what is left are terms of 0.125 to 0.875. A step of float32 sums cuts its 16 products and the sum so far at
    # 2^-23 of the largest at the worst: of 15 x 32768 in the codes' sums, of 32768 in the activations' (which the bias
    # multiplies). So a step of 16 columns adds at most 17 x 2^-23 (15 scale + |bias|) x 32768, and the group's end and the
    # sums of groups, all of them small, 2^-20 of the terms left.
    gen = gen_of(49)
    rows, tokens = 64, 4
    codes = torch.randint(0, 16, (rows, cols), device=cuda, generator=gen)
    x = (torch.randint(1, 8, (tokens, cols), device=cuda, generator=gen) / 8).half()
    for c in range(0, cols, 32):
        for at in (c, c + 4):
            codes[:, at + 1] = codes[:, at]
            x[:, at], x[:, at + 1] = 32768, -32768
    words = sum(codes.reshape(rows, -1, 8)[..., i] << (4 * i) for i in range(8))
    words = (words - ((words >> 31) << 32)).to(torch.int32)
    scales = (0.001 * (1 + torch.rand(rows, cols // group, device=cuda, generator=gen))).half()
    biases = (-7.5 * scales.float()).half()
    p = words, scales, biases
    w, mag = floats64(p)
    want = x.double() @ w.mT
    left = x.double().where(x.abs() < 1, 0.0)
    step = (15 * scales.double() + biases.double().abs()).sum(-1) * group / 16 * 17 * 32768 * 2.0**-23
    off = step + 2.0**-20 * (left @ mag.mT) + last(want, F16)
    assert (off < 0.05 * (left @ mag.mT)).all()
    close(affine.QuantizedLinear(*p, group_size=group)(x), want, off)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_wide_shared_expert_in_windows(cuda, dtype):
    # (9 and more tokens of 59 million weights are where the cost of gate and up in one launch passes that of a prompt's)
    gen = gen_of(50)
    hidden, ffn, group = 8192, 7680, 128
    s = [positive(gen, (), *d, group) for d in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
    mlp = affine.QuantizedMLP(*(affine.QuantizedLinear(*p, group_size=group) for p in s))
    x = positive_rows(gen, 16, hidden, dtype)
    each = torch.cat([mlp(x[i : i + 1]) for i in range(16)])
    for tokens in (2, 8, 9, 16):
        assert torch.equal(mlp(x[:tokens]), each[:tokens])
    h, eh = glu64(x, s[0], s[1], group, dtype)
    want, off = product64(h, s[2], group, dtype)
    near(each, want, off + eh @ floats64(s[2])[0].mT)


@pytest.mark.parametrize("ffn, tokens", [(4096, 500), (640, 2900)])
def test_gate_and_up_of_a_long_prompt_are_not_rounded_before_their_product(cuda, ffn, tokens):
    # gate rows of one negative value each take an activation row of one value to -11 .. -9, where float16 has steps of 2^-7
    # and silu follows them nearly in full (0.4 % at the most); up rows of one value to 480 .. 560; down is the identity.
    # Every weight is a float16 and every sum of 256 equal terms is off by 2^-24 a step at most, 2^-14 of itself in all by the
    # tensor core's 17 cuts a step of 16; silu's slope here is less than 12 times its value to one of the gate's.
    hidden, group = 256, 64
    gen = gen_of(51)

    def rows_of(values, rows, cols):
        codes = torch.zeros(rows, cols // 8, dtype=torch.int32, device=cuda)
        return codes, torch.zeros(rows, cols // group, dtype=F16, device=cuda), values.half()[:, None].expand(-1, cols // group).contiguous()

    gate = rows_of(-(9 + 2 * torch.rand(ffn, device=cuda, generator=gen)) / 256, ffn, hidden)
    up = rows_of((480 + 80 * torch.rand(ffn, device=cuda, generator=gen)) / 256, ffn, hidden)
    down = torch.zeros(hidden, ffn // 8, dtype=torch.int32, device=cuda)
    r = torch.arange(hidden, device=cuda)
    down[r, r // 8] = (1 << (4 * (r % 8))).to(torch.int32)
    down = down, torch.ones(hidden, ffn // group, dtype=F16, device=cuda), torch.zeros(hidden, ffn // group, dtype=F16, device=cuda)
    mlp = affine.QuantizedMLP(*(affine.QuantizedLinear(*p, group_size=group) for p in (gate, up, down)))
    assert mlp._apart(tokens)
    x = (1 + 0.03 * torch.rand(tokens, 1, device=cuda, generator=gen)).half().expand(-1, hidden)
    g, u = (x.double() @ floats64(p)[0].mT for p in (gate, up))
    want = (g * torch.sigmoid(g) * u)[:, :hidden]
    close(mlp(x), want, 2 * last(want, F16) + 13 * 2.0**-14 * want.abs())
    assert not affine.failed()


def small_block(gen, router_on="cuda", gate_on="cuda"):
    _, _, glu, mlp = positive_experts(gen, 8, 64, 64, 64, 32, 32)
    router = torch.randn(8, 64, device="cuda", generator=gen).half()
    sgate = torch.randn(1, 64, device="cuda", generator=gen).half()
    return fused.SparseMoeBlock(router.to(router_on), glu, mlp, sgate.to(gate_on), 2)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens", [1, 70])
def test_a_block_refuses_weights_of_the_route_on_another_device(cuda, dtype, tokens):
    gen = gen_of(52)
    x = torch.randn(tokens, 64, device=cuda, generator=gen).to(dtype)
    assert small_block(gen)(x).shape == x.shape
    for where in (dict(router_on="cpu"), dict(gate_on="cpu")):
        block = small_block(gen, **where)
        with pytest.raises(ValueError, match="CUDA|device"):
            block(x)
        for route in (fused.route, fused.route_window):
            if route is fused.route or (dtype == F16 and tokens <= 64):
                with pytest.raises(ValueError, match="CUDA|device"):
                    route(block.gate, block.shared_expert_gate, x, 2)


def test_a_route_refuses_activations_of_another_width(cuda):
    gen = gen_of(53)
    block = small_block(gen)
    for shape in ((1, 96), (2, 32), (1, 127)):
        x = torch.randn(*shape, device=cuda, generator=gen).half()
        for route in (fused.route_window, fused.route):
            with pytest.raises(ValueError, match="64"):
                route(block.gate, block.shared_expert_gate, x, 2)
        with pytest.raises(ValueError, match="64"):
            block(x)


def test_counters_for_captured_routes_are_zero_before_any_stream_can_use_them(cuda, monkeypatch):
    # (a first call on a busy stream makes them; a graph that is captured and replayed on another stream does not wait for it)
    block = small_block(gen_of(54))
    x = torch.randn(3, 64, device=cuda, generator=gen_of(55)).half()
    want = block(x)
    monkeypatch.setattr(fused, "_COUNTER_POOL", {})
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(busy):
        used = torch.ones(1 << 18, dtype=torch.int32, device=cuda)  # memory of their size that held something else
        assert used.any()  # (and the kernels loaded)
        torch.cuda.synchronize()
        del used
        torch.cuda._sleep(200_000_000)  # a tenth of a second
        assert not busy.query()
        block(x)
        seen = next(iter(fused._COUNTER_POOL.values()))[0]
    with torch.cuda.stream(other):
        assert not seen.any()
        assert torch.equal(block(x), want)
    torch.cuda.synchronize()


def test_eager_routes_on_several_streams_have_counters_of_their_own(cuda):
    gen = gen_of(56)
    block = small_block(gen)
    streams = [torch.cuda.Stream() for _ in range(4)]
    xs = [torch.randn(t, 64, device=cuda, generator=gen).half() for t in (1, 9, 33, 64)]
    want = [block(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for st, x in zip(streams, xs):
            with torch.cuda.stream(st):
                got.append(block(x))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("call", ["layer", "block", "prompt", "experts"])
def test_a_wait_that_runs_out_is_a_status_the_host_reads(cuda, call, dtype):
    # one copy of each launch never counts as landed; the launch ends, the status says so, and the next call is right again
    if dtype == F32 and call in ("prompt", "experts"):
        pytest.skip("float16 alone has a prompt's kernel")
    gen = gen_of(57)
    tokens, hidden = {"layer": 5, "block": 3, "prompt": 700, "experts": 1100}[call], 512
    _, s, glu, mlp = positive_experts(gen, 6, hidden, 256, 384, 64, 64)
    x = positive_rows(gen, tokens, hidden, dtype)
    idx = torch.randint(0, 6, (tokens, 2), dtype=torch.int32, device=cuda, generator=gen)
    w, g = torch.rand(tokens, 2, device=cuda, generator=gen), torch.randn(tokens, 1, device=cuda, generator=gen).to(dtype)
    wide = affine.QuantizedLinear(*positive(gen, (), 40, 16384, 64))  # (more copies to come behind the one that is missed)
    wide_x = positive_rows(gen, tokens, 16384, dtype)

    def run():
        if call == "block":
            return affine.moe(glu, mlp, x, idx, w, g)
        return glu(x, idx) if call == "experts" else mlp.gate_proj(x) if call == "prompt" else wide(wide_x)

    affine.failed(clear=True)
    want = run()
    assert not affine.failed()
    try:
        _lib.call("smoe_q4_wait_test", 1)
        run()
        assert affine.failed(clear=True)
    finally:
        _lib.call("smoe_q4_wait_test", 0)
    assert not affine.failed()
    assert torch.equal(run(), want) and not affine.failed()


@pytest.mark.parametrize("tokens", [0, 1, 5, 70, 600])
@pytest.mark.parametrize("which", ["shared", "routed"])
def test_a_block_of_gguf_experts_beside_4_bit_ones(cuda, which, tokens):
    # the shared expert 4-bit and the routed experts GGUF blocks (the reference's own mixture), and the other way round: the
    # blocks' part is taken as it comes, the 4-bit part by its definition, the combine's roundings counted one by one
    gen = gen_of(58)
    hidden, ffn, experts, k, group = 256, 512, 6, 2, 32
    rng = np.random.default_rng(5)

    def stack(*shape):
        data = Q.random_blocks("Q8_0", int(np.prod(shape)) // 32, rng, normal=0.001).reshape(-1)
        return torch.from_numpy(data).to(cuda), "Q8_0", shape

    r, s, glu, mlp = positive_experts(gen, experts, hidden, ffn, ffn, group, group)
    if which == "shared":
        glu = blocks.BlockSwitchGLU(*(blocks.BlockSwitchLinear(*stack(experts, *d)) for d in ((ffn, hidden), (ffn, hidden), (hidden, ffn))))
    else:
        mlp = blocks.BlockMLP(*(blocks.BlockLinear(*stack(*d)) for d in ((ffn, hidden), (ffn, hidden), (hidden, ffn))))
    router, sgate = (torch.randn(n, hidden, device=cuda, generator=gen).half() for n in (experts, 1))
    block = fused.SparseMoeBlock(router, glu, mlp, sgate, k)
    x = positive_rows(gen, tokens, hidden, F16)
    got = block(x)
    assert got.shape == x.shape and got.dtype == F16
    if not tokens:
        return
    idx, w, g = fused.route(block.gate, block.shared_expert_gate, x, k)
    idx, share, eps = idx.view(torch.int32).long(), torch.sigmoid(g.double()), 2.0**-11
    if which == "shared":
        y, ey = glu(x, idx.to(torch.int32)).double(), 0
        h, eh = glu64(x, s[0], s[1], group, F16, rounded=True)
        sh, es = product64(h, s[2], group, F16)
        es = es + (eh + eps * h) @ floats64(s[2])[0].mT
    else:
        sh, es = mlp(x).double(), 0
        y, ey = torch.zeros(2, tokens, k, hidden, dtype=torch.float64, device=cuda)
        for e in range(experts):
            t, j = (idx == e).nonzero(as_tuple=True)
            gate, up, down = ([a[e] for a in p] for p in r)
            h, eh = glu64(x[t], gate, up, group, F16, rounded=True)
            y[t, j], ey[t, j] = product64(h, down, group, F16)
            ey[t, j] += (eh + eps * h) @ floats64(down)[0].mT
    sums = (y * w.double()[..., None]).sum(1)
    want = sums + share * sh
    off = (1.01 * ey * w.double()[..., None]).sum(1) if which == "routed" else 0
    off = off + 2 * eps * sums.abs() + share * (1.01 * es + 4 * eps * sh.abs()) + eps * want.abs() + 2.0**-23
    close(got, want, off)


def test_a_4_bit_block_as_a_step_with_its_copies(cuda):
    gen = gen_of(59)
    block = small_block(gen)
    for tokens in (1, 17):
        x = torch.randn(tokens, 64, device=cuda, generator=gen).half()
        want = block(x)
        step = fused.GraphedBlock(block, tokens, 64, F16, cuda, host_io=True)
        for _ in range(2):
            out = step(x.cpu())
            step.ready.synchronize()
            assert torch.equal(out, want.cpu())


def alone(w, mag, dtype, rounded=False):
    """How far a weight may be that an activation of one brings out alone: the group's two terms in float32, its rounding."""
    return mag * 2.0**-22 + last(w, dtype) * (2 if rounded else 1)


@pytest.mark.parametrize("rows, cols, group", [(15, 96, 32), (16, 64, 64), (33, 160, 32), (129, 384, 128), (300, 1056, 32), (70, 2560, 64)])
@pytest.mark.parametrize("tokens", [1, 7, 16, 24, 200])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_every_weight_of_a_layer_alone(cuda, rows, cols, group, tokens, dtype):
    gen = gen_of(60 + tokens)
    p = parts(gen, (), rows, cols, group)
    layer = affine.QuantizedLinear(*p, group_size=group)
    w, mag = floats64(p)
    eye = torch.eye(cols, dtype=dtype, device=cuda)
    got = torch.cat([layer(eye[c : c + tokens]) for c in range(0, cols, tokens)]).T
    close(got, w, alone(w, mag, dtype, tokens > 16))


@pytest.mark.parametrize("experts, rows, cols, group", [(3, 33, 160, 32), (5, 130, 256, 64), (2, 16, 384, 128)])
@pytest.mark.parametrize("dtype, tiles", [(F16, False), (F16, True), (F32, False)])
def test_every_weight_of_a_stack_alone(cuda, experts, rows, cols, group, dtype, tiles, monkeypatch):
    gen = gen_of(61)
    p = parts(gen, (experts,), rows, cols, group)
    stack = affine.QuantizedSwitchLinear(*p, group_size=group)
    monkeypatch.setattr(affine, "_by_tiles", lambda lin, dt, pairs: tiles)
    w, mag = floats64(p)
    idx = torch.stack([torch.randperm(experts, device=cuda, generator=gen) for _ in range(cols)]).to(torch.int32)
    got = stack(torch.eye(cols, dtype=dtype, device=cuda)[:, None, None], idx)[:, :, 0]  # (cols, experts, rows)
    want, mag = (t.permute(2, 0, 1).gather(1, idx.long()[..., None].expand(-1, -1, rows)) for t in (w, mag))
    close(got, want, alone(want, mag, dtype, tiles))


@pytest.mark.parametrize("rows, cols, group", SHAPES)
@pytest.mark.parametrize("tokens", [1, 5, 8, 13, 16, 17, 48, 700])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_a_layer_of_positive_weights(cuda, rows, cols, group, tokens, dtype):
    gen = gen_of(rows + cols + tokens)
    p = positive(gen, (), rows, cols, group)
    x = positive_rows(gen, tokens, cols, dtype)
    near(affine.QuantizedLinear(*p, group_size=group)(x), *layer64(x, p, group, dtype))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens, k, experts, hidden, ffn, shared, group, down_group",
                         [(300, 8, 17, 320, 160, 96, 32, 32), (700, 4, 5, 256, 384, 640, 128, 64), (260, 10, 12, 1024, 64, 2048, 64, 64),
                          (70, 32, 64, 96, 64, 64, 32, 64), (2100, 1, 1, 64, 128, 64, 64, 64), (1100, 3, 1500, 64, 32, 32, 32, 32)])
def test_a_prompt_of_positive_weights(cuda, dtype, tokens, k, experts, hidden, ffn, shared, group, down_group):
    gen = gen_of(tokens + k)
    r, s, glu, mlp = positive_experts(gen, experts, hidden, ffn, shared, group, down_group)
    x = positive_rows(gen, tokens, hidden, dtype)
    w = 0.05 + torch.rand(tokens, k, device=cuda, generator=gen)
    g = torch.randn(tokens, 1, device=cuda, generator=gen).to(dtype)
    idx = torch.randint(0, experts, (tokens, k), dtype=torch.int32, device=cuda, generator=gen)
    idx[::5, 0], idx[7] = experts, -1
    near(affine.moe(glu, mlp, x, idx, w, g), *moe64(x, r, s, idx, w, g, group, down_group, dtype, rounded=dtype == F16))
    assert not affine.failed()


@pytest.mark.parametrize("rows, cols, group", [(1, 32, 32), (130, 96, 32), (300, 1024, 128), (1000, 320, 64)])
@pytest.mark.parametrize("tokens", [1, 7, 16, 33, 161, 600])
def test_the_prompts_kernel_at_any_count_in_both_types(cuda, rows, cols, group, tokens):
    gen = gen_of(rows + tokens)
    p = positive(gen, (), rows, cols, group)
    layer = affine.QuantizedLinear(*p, group_size=group)
    x = positive_rows(gen, tokens, cols, F16)
    want, off = product64(x, p, group)
    off = off + x.double() @ last(floats64(p)[0], F16).mT
    got = layer._prompt(x)
    assert got.dtype == F32
    near(got, want, off + last(want, F32))
    half = torch.full((tokens + 1, rows), 7.0, dtype=F16, device=cuda)
    _lib.call("smoe_q4_prompt", layer.data_ptr, rows, cols, group, x.data_ptr(), tokens, half.data_ptr(), _lib.F16, _lib.stream())
    assert torch.equal(half[:-1], got.half()) and (half[-1] == 7).all()


def test_a_windows_route_with_a_gate_of_either_type(cuda):
    gen = gen_of(62)
    block = small_block(gen)
    for tokens in (1, 8, 13, 64):
        x = torch.randn(tokens, 64, device=cuda, generator=gen).half()
        idx, w, g = fused.route_window(block.gate, block.shared_expert_gate, x, 2)
        idx32, w32, g32 = fused.route_window(block.gate, block.shared_expert_gate, x, 2, torch.float32)
        assert torch.equal(idx, idx32) and torch.equal(w, w32) and g.dtype == F16 and torch.equal(g32.half(), g)
        want = x.double() @ block.shared_expert_gate.weight.double().mT
        close(g32, want, 64 * 2.0**-23 * (x.double().abs() @ block.shared_expert_gate.weight.double().abs().mT))
    assert fused.route_window(block.gate, block.shared_expert_gate, x, 2, torch.bfloat16) is None


def test_prompts_blocks_and_a_graph_on_several_streams(cuda):
    gen = gen_of(63)
    _, s, glu, mlp = positive_experts(gen, 9, 512, 256, 1024, 64, 64)
    router, sgate = (torch.randn(n, 512, device=cuda, generator=gen).half() for n in (9, 1))
    block = fused.SparseMoeBlock(router, glu, mlp, sgate, 3)
    xs = [positive_rows(gen, t, 512, F16) for t in (900, 64, 1000, 800)]
    idx = torch.randint(0, 9, (900, 3), dtype=torch.int32, device=cuda, generator=gen)
    step = fused.GraphedBlock(block, 800, 512, F16, cuda)
    calls = [lambda x: glu(x, idx), block, mlp.gate_proj, step]
    want = [call(x).clone() for call, x in zip(calls, xs)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(30):
        got = []
        for st, call, x in zip(streams, calls, xs):
            with torch.cuda.stream(st):
                got.append(call(x))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert not affine.failed()
