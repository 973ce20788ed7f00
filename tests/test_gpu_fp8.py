"""The kernels of 8-bit linear layers against their formulas in 64 bits.

Bounds.  e4m3 has a step of 2^(e - 3) for a magnitude in [2^e, 2^(e + 1)), of 2^-9 below 2^-6, and a rounding is off by half a step: at
most max(2^-4 |t|, 2^-10) for a value t.  u = 2^-24 is a float32 rounding.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
LEAST = 448.0 * 2.0 ** -126
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def kblocks(n):
    return -(-n // 128)


def rnd(*shape, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV) * scale


def spread(scales, rows, t, k):
    return scales.repeat_interleave(rows, 0)[:t].repeat_interleave(128, 1)[:, :k]


def block_max(x, rows):
    t, k = x.shape
    p = x.new_zeros(kblocks(t) * 128 if rows == 128 else t, kblocks(k) * 128)
    p[:t, :k] = x.abs()
    return p.view(-1, rows, kblocks(k), 128).amax(dim=(1, 3))


def check_quantized(q, scales, y, rows, rel):
    """q and scales stand for y (float64), which the kernel knows up to rel (a number, or one for each value) of each value."""
    amax = block_max(y, rows)
    want = amax.clamp(min=LEAST) / 448.0
    assert torch.isfinite(scales).all() and torch.isfinite(q.float()).all()
    worst = float(rel) if not torch.is_tensor(rel) else None
    off = (block_max(y.abs() * rel, rows) / 448.0 if worst is None else worst * want) + 2 * U * want
    assert ((scales.double() - want).abs() <= off).all()
    s = spread(scales.double(), rows, *y.shape)
    t = (y / s).abs()
    # the rounding to 8 bits, what y itself is off by, and two roundings of 448 / a and its product
    assert ((q.double() * s - y).abs() <= s * torch.clamp(t * (1 + 4 * U) * 2.0 ** -4, min=2.0 ** -10) + y.abs() * (rel + 4 * U) * 1.0625).all()


def plain_quantize(x, rows):
    """The same formula in float32, rounded by torch: the same bits (quotients of tensors: torch makes a quotient with a number
    a product with the reciprocal)."""
    a = block_max(x.float(), rows).clamp(min=LEAST)
    top = torch.full_like(a, 448.0)
    return (x.float() * spread(top / a, rows, *x.shape)).to(torch.float8_e4m3fn), a / top


SIZES = [(1, 1), (1, 128), (3, 127), (2, 129), (5, 264), (128, 256), (129, 1000), (300, 4096), (257, 131), (131, 1002), (6, 262)]


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,K", SIZES)
def test_quantize(T, K, dtype, rows):
    from purhie_b200.csrc import fp8
    x = rnd(T, K, seed=T + K, scale=5.0).to(DT[dtype])
    x[T // 2] = 0
    q, s = fp8.quantize(x, block_rows=rows)
    check_quantized(q, s, x.double(), rows, 0.0)
    wq, ws = plain_quantize(x, rows)
    assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, ws)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("off,stride", [(0, 1040), (8, 1040), (2, 1040), (2, 1002), (1, 1040), (8, 1003)])
def test_quantize_of_strided_rows(off, stride, rows):
    from purhie_b200.csrc import fp8
    held = rnd(200, stride, seed=1).to(torch.bfloat16)
    x = held[:, off:off + 520]
    q, s = fp8.quantize(x, block_rows=rows)
    wq, ws = plain_quantize(x, rows)
    assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, ws)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_extremes(rows):
    """Zeros, the smallest and largest numbers, and each kind of number that is none: a block keeps what it was."""
    from purhie_b200.csrc import fp8
    x = torch.zeros(256, 512, device=DEV)
    x[0, 0:128] = 1e-44
    x[0, 128:256] = torch.finfo(torch.float32).max
    x[0, 300] = float("nan")
    x[0, 400] = float("-inf")
    x[0, 401] = 2.0
    q, s = fp8.quantize(x, block_rows=rows)
    wq, ws = plain_quantize(x, rows)
    # torch's amax keeps what is not a number, and so do the products
    assert torch.equal(torch.nan_to_num(s, nan=-1.0), torch.nan_to_num(ws, nan=-1.0))
    assert torch.equal(torch.nan_to_num(q.float(), nan=-1.0), torch.nan_to_num(wq.float(), nan=-1.0))
    assert torch.isnan(s[0, 2]) and torch.isinf(s[0, 3]) and s[-1, 0] == 2.0 ** -126


def test_quantize_writes_only_its_own():
    from purhie_b200.csrc import fp8
    x = rnd(7, 1000, seed=3)
    held_q = torch.full((9, 1000), 1.0, device=DEV).to(torch.float8_e4m3fn)
    held_s = torch.full((9, 8), -5.0, device=DEV)
    fp8.quantize(x, held_q[1:8], held_s[1:8])
    assert (held_q[0].float() == 1).all() and (held_q[8].float() == 1).all() and (held_s[0] == -5).all() and (held_s[8] == -5).all()


def test_rows_past_two_to_the_31():
    """An offset of more than 2^31 values, in front of and behind."""
    from purhie_b200.csrc import fp8
    held = torch.zeros(3, 2 ** 30 + 512, dtype=torch.bfloat16, device=DEV)
    x = held[:, :640]
    x.copy_(rnd(3, 640, seed=4).to(torch.bfloat16))
    q, s = fp8.quantize(x)
    wq, ws = plain_quantize(x.contiguous(), 1)
    assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, ws)


@pytest.mark.parametrize("E", [1, 64, 127, 128, 1000, 1002, 2056, 4096, 5120, 8200, 16400, 32768])
@pytest.mark.parametrize("add,parts", [(None, 1), ("f32", 1), ("bf16", 1), ("f32", 3), ("f32", 9), ("bf16", 7)])
def test_add_rmsnorm(E, add, parts):
    from purhie_b200.csrc import fp8
    T, eps = 5, 1e-5
    x = rnd(T, E, seed=E, scale=3.0)
    x[2] = 0
    a = None if add is None else rnd(parts, T, E, seed=E + 1).to(DT[add])
    if a is not None:
        a[:, 2] = 0
    w = 1 + 0.3 * rnd(E, seed=2)
    v = x.double() if a is None else x.double() + a.double().sum(0)
    size = x.abs().double() if a is None else x.abs().double() + a.abs().double().sum(0)
    out = torch.empty(T, E, device=DEV)
    q, s = fp8.add_rmsnorm(x, None if a is None else a.view(parts, T, E) if parts > 1 else a[0], w, eps, add_splits=parts, x_out=out)
    v_off = parts * U * size                                                     # each addition rounds once
    assert ((out.double() - v).abs() <= v_off).all()
    # the kernel's own v, exactly known; a sum of squares over 8 U values a thread, five exchanges and five more: at most 64 + 10
    # roundings up and down the tree, each square one; the root's and the two products' few
    v = out.double()
    y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.double()
    check_quantized(q, s, y, 1, 100 * U)


@pytest.mark.parametrize("E", [1000, 5120, 5248, 8320])
@pytest.mark.parametrize("parts", [2, 5, 9, 13])
def test_a_row_s_norm_does_not_depend_on_the_others(parts, E):
    """More rows than multiprocessors and few: the same bits."""
    from purhie_b200.csrc import fp8
    T = 2 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    x, a, w = rnd(T, E, seed=E), rnd(parts, T, E, seed=parts), 1 + 0.3 * rnd(E, seed=2)
    out = torch.empty_like(x)
    q, s = fp8.add_rmsnorm(x, a, w, 1e-6, add_splits=parts, x_out=out)
    v = x.clone()
    for i in range(parts):
        v += a[i]
    assert torch.equal(out, v)
    few = torch.empty(3, E, device=DEV)
    q1, s1 = fp8.add_rmsnorm(x[7:10].contiguous(), a[:, 7:10].contiguous(), w, 1e-6, add_splits=parts, x_out=few)
    assert torch.equal(few, out[7:10]) and torch.equal(q1.view(torch.uint8), q[7:10].view(torch.uint8)) and torch.equal(s1, s[7:10])


def test_add_rmsnorm_keeps_the_sum_where_told():
    from purhie_b200.csrc import fp8
    x, a, w = rnd(6, 512, seed=1), rnd(6, 512, seed=2), torch.ones(512, device=DEV)
    before = x.clone()
    q0, s0 = fp8.add_rmsnorm(x, a, w, 1e-6, write_x=False)
    assert torch.equal(x, before)
    rows = torch.tensor([5, 0, 0, -1, 6, 3], dtype=torch.int32, device=DEV)
    held_q, held_s = torch.full((6, 512), 3.0, device=DEV).to(torch.float8_e4m3fn), torch.full((6, 4), 7.0, device=DEV)
    q1, s1 = fp8.add_rmsnorm(x, a, w, 1e-6, held_q, held_s, rows=rows)
    assert torch.equal(x, before)
    for r, t in enumerate(rows.tolist()):
        if 0 <= t < 6:
            assert torch.equal(q1[r].view(torch.uint8), q0[t].view(torch.uint8)) and torch.equal(s1[r], s0[t])
        else:
            assert (q1[r].float() == 3.0).all() and (s1[r] == 7.0).all()
    q2, s2 = fp8.add_rmsnorm(x, a, w, 1e-6)
    assert torch.equal(x, before + a) and torch.equal(q2.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s2, s0)


def gate_value(g, u, gate):
    """The gated activation in 64 bits, and the argument of its exponential."""
    if gate is None:
        arg, num, up = -g, g, u
    elif gate == "gelu_tanh":
        arg, num, up = -2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3), g, u
    else:
        alpha, limit, shift = gate
        num, up = g.clamp(max=limit), u.clamp(-limit, limit) + shift
        arg = -alpha * num
    return num * torch.sigmoid(-arg) * up, arg, num, up


@pytest.mark.parametrize("gate", [None, (1.702, 7.0, 1.0), "gelu_tanh"])
@pytest.mark.parametrize("dtype,parts", [("f32", 1), ("bf16", 1), ("f32", 3), ("f32", 7), ("bf16", 4)])
@pytest.mark.parametrize("T,F", [(1, 1), (3, 127), (2, 128), (5, 1000), (4, 1001), (7, 1002), (33, 4104)])
def test_gated(T, F, dtype, parts, gate):
    from purhie_b200.csrc import fp8
    gu = rnd(parts, T, 2 * F, seed=T + F, scale=4.0).to(DT[dtype])
    q, s = fp8.gated(gu if parts > 1 else gu[0], splits=parts, gate=gate)
    both = gu[0].float()
    for i in range(1, parts):
        both = both + gu[i].float()                       # the kernel's own order, so that both sides gate the same numbers
    h, arg, num, up = gate_value(both[:, 0::2].double(), both[:, 1::2].double(), gate)
    # an exponential whose argument is a few roundings off, its own two units, a quotient of two units, the products; with the
    # quotient's denominator past 2^126 the result is zero
    rel = (24 + 8 * arg.abs().clamp(max=90)) * U
    tiny = (num * up).abs() * 2.0 ** -125
    rel = rel + tiny / h.abs().clamp(min=1e-300)
    check_quantized(q, s, h, 1, rel)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("F", [1000, 1002, 1001])
@pytest.mark.parametrize("T", [3, 5200])
def test_inputs_off_their_boundaries(T, F, dtype):
    """Rows that start one, two and four values behind a boundary, few and many of them, give what aligned ones give."""
    from purhie_b200.csrc import fp8
    gu, x, ones = rnd(T, 2 * F, seed=F, scale=3.0).to(DT[dtype]), rnd(T, F, seed=F + 1).to(DT[dtype]), torch.ones(F, device=DEV)
    want_g, want_x, want_n = fp8.gated(gu), fp8.quantize(x), fp8.add_rmsnorm(x.float(), x, ones, 1e-6, write_x=False)
    for off in (1, 2, 4):
        def moved(t):
            y = torch.empty(t.numel() + 8, dtype=t.dtype, device=DEV)[off:off + t.numel()].view(t.shape)
            return y.copy_(t)
        for got, want in ((fp8.gated(moved(gu)), want_g), (fp8.quantize(moved(x)), want_x)):
            assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
        # a row's sum of squares is added up in another order: its factor is some roundings off, and a value may fall to its neighbour
        q, s = fp8.add_rmsnorm(moved(x.float()), moved(x), ones, 1e-6, write_x=False)
        assert ((s - want_n[1]).abs() <= 100 * U * s).all()
        assert ((q.float() - want_n[0].float()).abs() <= want_n[0].float().abs().clamp(min=2.0 ** -6) * 2.0 ** -3).all()


def test_gated_keeps_what_is_not_a_number():
    from purhie_b200.csrc import fp8
    gu = rnd(2, 512, seed=1)
    gu[0, 4] = float("nan")
    gu[1, 301] = float("inf")
    for gate in (None, (1.702, 7.0, 1.0), "gelu_tanh"):
        q, s = fp8.gated(gu, gate=gate)
        assert torch.isnan(s[0, 0]) and torch.isfinite(s[0, 1]) and torch.isfinite(s[1, 0])
        assert torch.isinf(s[1, 1]) if not isinstance(gate, tuple) else torch.isfinite(s[1, 1])


def operands(M, N, K, seed):
    """e4m3 values over the whole range with scales far apart, so that a wrong scale is not a small error."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(M, K, generator=g, device=DEV) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = (torch.randn(N, K, generator=g, device=DEV) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    xs = torch.exp(torch.randn(M, kblocks(K), generator=g, device=DEV) * 1.5)
    ws = torch.exp(torch.randn(kblocks(N), kblocks(K), generator=g, device=DEV) * 1.5)
    return x, xs, w, ws


def check_product(out, x, xs, w, ws):
    M, K = x.shape
    N = w.shape[0]
    a, b = x.double() * spread(xs.double(), 1, M, K), w.double() * spread(ws.double(), 128, N, K)
    want, size = a @ b.T, a.abs() @ b.abs().T
    # at most K additions of exact products and one multiply-add per block of K and split, each off by a unit (the tensor cores
    # may cut where float32 arithmetic rounds); the scales' product rounds once
    off = (K + kblocks(K) + 12) * 2 * U * size + want.abs() * torch.finfo(out.dtype).eps / 2
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() <= off).all()


SHAPES = [(1, 16), (64, 128), (100, 48), (129, 144), (257, 272), (1000, 2064), (2304, 512)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 65, 96, 97, 128, 129, 300])
def test_product(M, N, K, out):
    from purhie_b200.csrc import fp8
    x, xs, w, ws = operands(M, N, K, M + N + K)
    y = fp8.gemm(x, xs, w, ws, out_dtype=DT[out])
    check_product(y, x, xs, w, ws)
    fp8.check_errors()


@pytest.mark.parametrize("tile,splits", [(t, s) for t in (16, 32, 64, 96, 256) for s in (1, 2, 3, 7, 16)])
@pytest.mark.parametrize("M,N", [(1, 200), (40, 200), (150, 200), (290, 515)])
def test_product_of_every_tile_and_split(M, N, splits, tile):
    """Small whole numbers and scales that are powers of two: every sum is exact in float32, so every variant gives the same bits."""
    from purhie_b200.csrc import fp8
    K = 2064
    g = torch.Generator(device=DEV).manual_seed(splits)
    x = torch.randint(-4, 5, (M, K), generator=g, device=DEV).float().to(torch.float8_e4m3fn)
    w = torch.randint(-4, 5, (N, K), generator=g, device=DEV).float().to(torch.float8_e4m3fn)
    xs = torch.exp2(torch.randint(-2, 3, (M, kblocks(K)), generator=g, device=DEV).float())
    ws = torch.exp2(torch.randint(-2, 3, (kblocks(N), kblocks(K)), generator=g, device=DEV).float())
    want = (x.double() * spread(xs.double(), 1, M, K)) @ (w.double() * spread(ws.double(), 128, N, K)).T
    held = torch.full((splits + 2, M, N), -7.0, device=DEV)
    if splits > 1:
        fp8.gemm(x, xs, w, ws, held[1:splits + 1], tile=tile, splits=splits)
        assert torch.equal(held[1:splits + 1].double().sum(0), want)
    else:
        fp8.gemm(x, xs, w, ws, held[1], tile=tile, splits=1)
        assert torch.equal(held[1].double(), want)
    assert (held[0] == -7).all() and (held[splits + 1] == -7).all()
    for dtype in DT.values():
        assert torch.equal(fp8.gemm(x, xs, w, ws, out_dtype=dtype, tile=tile), want.to(dtype))
    fp8.check_errors()


def test_product_into_places_off_their_boundaries():
    """Outputs that start on their own type's boundary only, at widths whose rows would allow vectors."""
    from purhie_b200.csrc import fp8
    for M, N, K, tile in ((3, 260, 1040, 16), (70, 132, 2064, 64), (90, 132, 2064, 96), (300, 264, 400, 256)):
        x, xs, w, ws = operands(M, N, K, M)
        for dtype in DT.values():
            held = torch.zeros(M * N + 9, dtype=dtype, device=DEV)
            y = held[1:M * N + 1].view(M, N)
            for splits in (0, 1):
                y.fill_(float("nan"))
                fp8.gemm(x, xs, w, ws, y, tile=tile, splits=splits)
                check_product(y, x, xs, w, ws)
            assert held[0] == 0 and (held[M * N + 1:] == 0).all()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(256, 256, 128), (257, 264, 16), (1000, 1003, 656), (2100, 2304, 1040), (2048, 4104, 512), (5000, 1024, 400)])
def test_product_on_pairs(M, N, K, out):
    """More tiles than pairs and fewer, outputs that the copy engine stores and such that the threads store."""
    from purhie_b200.csrc import fp8
    x, xs, w, ws = operands(M, N, K, M + N + K)
    check_product(fp8.gemm(x, xs, w, ws, out_dtype=DT[out], tile=256), x, xs, w, ws)
    fp8.check_errors()


@pytest.mark.parametrize("gate", [None, (1.702, 7.0, 1.0), "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(1, 256, 16), (255, 768, 272), (300, 512, 2064), (1000, 2304, 656), (2100, 5120, 400)])
def test_product_with_the_activation(M, N, K, gate):
    """The fused form is the product on pairs and the activation of its float32 values: more tiles than pairs and fewer, rows that end
    inside a tile."""
    from purhie_b200.csrc import fp8
    x, xs, w, ws = operands(M, N, K, M + N + K)
    xs *= 0.01
    ws *= 0.01
    y = fp8.gemm(x, xs, w, ws, out_dtype=torch.float32, tile=256, splits=1)
    held_q, held_s = torch.full((M + 2, N // 2), 3.0, device=DEV).to(torch.float8_e4m3fn), torch.full((M + 2, N // 256), -1.0, device=DEV)
    q, s = fp8.gemm_gated(x, xs, w, ws, held_q[1:M + 1], held_s[1:M + 1], gate=gate)
    want_q, want_s = fp8.gated(y, gate=gate)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
    for i in (0, M + 1):
        assert (held_q[i].float() == 3).all() and (held_s[i] == -1).all()
    h, arg, num, up = gate_value(y[:, 0::2].double(), y[:, 1::2].double(), gate)
    rel = (24 + 8 * arg.abs().clamp(max=90)) * U + (num * up).abs() * 2.0 ** -125 / h.abs().clamp(min=1e-300)
    check_quantized(q, s, h, 1, rel)
    fp8.check_errors()


def test_product_with_the_activation_keeps_what_is_not_a_number():
    from purhie_b200.csrc import fp8
    x, xs, w, ws = operands(300, 512, 256, 1)
    xs *= 0.01
    ws *= 0.01
    xs[7, 1] = float("nan")
    xs[290, 0] = float("inf")
    q, s = fp8.gemm_gated(x, xs, w, ws)
    assert torch.isnan(s[7]).all() and not torch.isfinite(s[290]).any()
    fine = torch.ones(300, dtype=torch.bool, device=DEV)
    fine[7] = fine[290] = False
    assert torch.isfinite(s[fine]).all() and torch.isfinite(q[fine].float()).all()


def test_product_refusals():
    from purhie_b200.csrc import fp8
    from purhie_b200.native import KernelError
    x, xs, w, ws = operands(4, 64, 144, 1)
    with pytest.raises(KernelError, match="multiple of 16"):
        fp8.gemm(x[:, :136].contiguous(), xs, w[:, :136].contiguous(), ws)
    for splits in (3, 17):
        with pytest.raises(KernelError, match="parts of K"):
            fp8.gemm(x, xs, w, ws, tile=16, splits=splits)
    with pytest.raises(KernelError, match="negative"):
        fp8.gemm(x, xs, w, ws, splits=-1)
    with pytest.raises(KernelError, match="tile"):
        fp8.gemm(x, xs, w, ws, tile=48)
    with pytest.raises(KernelError, match="unsupported dtype"):
        fp8.gemm(x, xs, w, ws, out_dtype=torch.float16)
    with pytest.raises(KernelError, match="out must"):
        fp8.gemm(x, xs, w, ws, torch.empty(4, 63, device=DEV))
    with pytest.raises(KernelError, match="aligned"):
        held = torch.zeros(4 * 144 + 1, device=DEV).to(torch.float8_e4m3fn)
        fp8.gemm(held[1:].view(4, 144), xs, w, ws)
    with pytest.raises(KernelError, match="unsupported dtype"):
        fp8.quantize(torch.zeros(4, 4, dtype=torch.float16, device=DEV))
    with pytest.raises(KernelError, match="device"):
        fp8.quantize(torch.zeros(4, 4, device=DEV), scales=torch.zeros(4, 1))


def test_no_rows():
    from purhie_b200.csrc import fp8
    x, xs, w, ws = operands(4, 64, 144, 1)
    assert fp8.gemm(x[:0], xs[:0], w, ws).shape == (0, 64)
    q, s = fp8.quantize(torch.zeros(0, 300, device=DEV))
    assert q.shape == (0, 300) and s.shape == (0, 3)
    q, s = fp8.gated(torch.zeros(0, 600, device=DEV))
    assert q.shape == (0, 300) and s.shape == (0, 3)
    q, s = fp8.add_rmsnorm(torch.zeros(0, 300, device=DEV), None, torch.ones(300, device=DEV), 1e-6)
    assert q.shape == (0, 300) and s.shape == (0, 3)


def feed_forward(x, add, norm, gate_up, gate_up_s, down, down_s, early_w=False):
    from purhie_b200.csrc import fp8
    q, s = fp8.add_rmsnorm(x, add, norm, 1e-6, x_out=torch.empty_like(x))
    y = fp8.gemm(q, s, gate_up, gate_up_s, out_dtype=torch.float32, early_w=early_w)
    q2, s2 = fp8.gated(y)
    return fp8.gemm(q2, s2, down, down_s, out_dtype=torch.float32, early_w=early_w), (q, s, y, q2, s2)


def weights(E, F):
    from purhie_b200.csrc import fp8
    return (1 + 0.2 * rnd(E, seed=1), *fp8.quantize(rnd(2 * F, E, seed=2, scale=E ** -0.5).to(torch.bfloat16), block_rows=128),
            *fp8.quantize(rnd(E, F, seed=3, scale=F ** -0.5).to(torch.bfloat16), block_rows=128))


@pytest.mark.parametrize("T", [1, 9, 70, 200])
def test_feed_forward(T):
    """The operators one behind the other, each held to what the one in front gave."""
    E, F = 416, 1040
    w = weights(E, F)
    x, add = rnd(T, E, seed=4), rnd(T, E, seed=5).to(torch.bfloat16)
    out, (q, s, y, q2, s2) = feed_forward(x, add, *w)
    v = (x + add.float()).double()
    check_quantized(q, s, v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w[0].double(), 1, 100 * U)
    check_product(y, q, s, w[1], w[2])
    h, arg, _, _ = gate_value(y[:, 0::2].double(), y[:, 1::2].double(), None)
    check_quantized(q2, s2, h, 1, (24 + 8 * arg.abs()) * U)
    check_product(out, q2, s2, w[3], w[4])


def test_feed_forward_in_graphs_and_streams():
    """Captured and replayed on new inputs, twice over for two graphs at once, and on a stream of its own: the same bits."""
    from purhie_b200.csrc import fp8
    E, F, T = 416, 1040, 24
    w = weights(E, F)
    held = [(torch.zeros(T, E, device=DEV), torch.zeros(T, E, device=DEV).to(torch.bfloat16)) for _ in range(2)]
    inputs = [(rnd(T, E, seed=10 + i), rnd(T, E, seed=20 + i).to(torch.bfloat16)) for i in range(4)]
    want = [feed_forward(*i, *w)[0].clone() for i in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(4):
            assert torch.equal(feed_forward(*inputs[i], *w, early_w=True)[0], want[i])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = feed_forward(*h, *w, early_w=True)[0]
        graphs.append((g, out))
    for i in range(0, 4, 2):
        for j in range(2):
            held[j][0].copy_(inputs[i + j][0])
            held[j][1].copy_(inputs[i + j][1])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                graphs[j][0].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(graphs[j][1], want[i + j])
    fp8.check_errors()


def test_many_rows_in_graphs_and_streams():
    """The same for rows enough for pairs of CTAs, the activation in the first product's epilogue."""
    from purhie_b200.csrc import fp8
    E, F, T = 416, 1024, 700
    norm, up, up_s, down, down_s = weights(E, F)

    def run(x, add):
        q, s = fp8.add_rmsnorm(x, add, norm, 1e-6, x_out=torch.empty_like(x))
        q2, s2 = fp8.gemm_gated(q, s, up, up_s)
        return fp8.gemm(q2, s2, down, down_s, out_dtype=torch.float32, tile=256)
    inputs = [(rnd(T, E, seed=10 + i), rnd(T, E, seed=20 + i).to(torch.bfloat16)) for i in range(4)]
    want = [run(*i).clone() for i in inputs]
    held = [(torch.zeros(T, E, device=DEV), torch.zeros(T, E, device=DEV).to(torch.bfloat16)) for _ in range(2)]
    graphs = []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(*h)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(0, 4, 2):
        for j in range(2):
            held[j][0].copy_(inputs[i + j][0])
            held[j][1].copy_(inputs[i + j][1])
        torch.cuda.synchronize()
        for _ in range(3):
            for j in range(2):
                with torch.cuda.stream(streams[j]):
                    graphs[j][0].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(graphs[j][1], want[i + j])
    fp8.check_errors()


def test_plain_calls_and_checked_ones_are_the_same():
    """A call without outputs takes the compiled step, one with them the checks of the face: the same launches."""
    from purhie_b200.csrc import fp8, ops
    x, a, w, gu = rnd(9, 264, seed=1), rnd(2, 9, 264, seed=2), 1 + 0.1 * rnd(264, seed=3), rnd(9, 528, seed=4).to(torch.bfloat16)

    def outs(t, k, rows=1):
        return torch.empty(t, k, device=DEV).to(torch.float8_e4m3fn), torch.empty(kblocks(t) if rows > 1 else t, kblocks(k), device=DEV)

    def same(p, q):
        return torch.equal(p[0].view(torch.uint8), q[0].view(torch.uint8)) and torch.equal(p[1], q[1])
    before = ops.launches
    for rows in (1, 128):
        assert same(fp8.quantize(x, block_rows=rows), fp8.quantize(x, *outs(9, 264, rows), block_rows=rows))
    assert same(fp8.gated(gu), fp8.gated(gu, *outs(9, 264)))
    for parts, add in ((2, a), (1, a[0]), (1, a[:1]), (1, None)):
        y, z = x.clone(), x.clone()
        assert same(fp8.add_rmsnorm(y, add, w, 1e-6, add_splits=parts), fp8.add_rmsnorm(z, add, w, 1e-6, *outs(9, 264), add_splits=parts))
        assert torch.equal(y, z) and torch.equal(y, x) == (add is None)
    assert ops.launches == before + 14
    xq, xs, wq, ws = operands(9, 200, 2064, 5)
    for dtype in DT.values():
        assert torch.equal(fp8.gemm(xq, xs, wq, ws, out_dtype=dtype), fp8.gemm(xq, xs, wq, ws, torch.empty(9, 200, dtype=dtype, device=DEV)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), ops.on_current_stream():
        with torch.cuda.stream(torch.cuda.default_stream()):
            q = fp8.quantize(x)                      # the scope's stream is the side stream, whatever is current inside it
    side.synchronize()
    assert same(q, fp8.quantize(x))
