"""The Python faces where the stream of their scope is not the current one: what they allocate belongs to the stream that the launch
goes to."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def operands(M, N, K, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    blocks = lambda n: -(-n // 128)  # noqa: E731
    return ((torch.randn(M, K, generator=g, device=DEV) * 60).to(torch.float8_e4m3fn), 1 + torch.rand(M, blocks(K), generator=g, device=DEV),
            (torch.randn(N, K, generator=g, device=DEV) * 60).to(torch.float8_e4m3fn), 1 + torch.rand(blocks(N), blocks(K), generator=g, device=DEV))


def calls():
    """Each face that makes tensors of its own, plain and through the checks, and what it gives."""
    from purhie_b200.csrc import fp8, ops
    x, xs, w, ws = operands(24, 4096, 2304, 1)
    rows = torch.randn(24, 2304, device=DEV)
    norm = torch.ones(2304, device=DEV)
    out = torch.empty(24, 4096, device=DEV)
    q = torch.empty(24, 2304, dtype=torch.float8_e4m3fn, device=DEV)
    tile, parts = fp8.plan(24, 4096, 2304)
    assert parts > 1                                         # (room for the parts of K)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    gru = [torch.randn(1, 40, 48, device=DEV), torch.zeros(16, device=DEV), torch.zeros(16, device=DEV), torch.zeros(1, 16, device=DEV), i32(0, 40), i32(0),
           torch.empty(40, 16, device=DEV)]
    y = torch.empty(24, 2304, dtype=torch.bfloat16, device=DEV)
    return {
        "gemm": lambda: fp8.gemm(x, xs, w, ws),
        "gemm float32": lambda: fp8.gemm(x, xs, w, ws, out_dtype=torch.float32),
        "gemm into out": lambda: fp8.gemm(x, xs, w, ws, out),
        "gemm with a tile": lambda: fp8.gemm(x, xs, w, ws, tile=tile),
        "gemm in parts": lambda: fp8.gemm(x, xs, w, ws, splits=3),
        "gemm_gated": lambda: fp8.gemm_gated(x, xs, w, ws),
        "quantize": lambda: fp8.quantize(rows),
        "quantize into out": lambda: fp8.quantize(rows, q),
        "add_rmsnorm": lambda: fp8.add_rmsnorm(rows, None, norm, 1e-6),
        "add_rmsnorm into out": lambda: fp8.add_rmsnorm(rows, None, norm, 1e-6, q),
        "gated": lambda: fp8.gated(rows),
        "gated gelu": lambda: fp8.gated(rows, gate="gelu_tanh"),
        "add_weight_sumsq": lambda: ops.add_weight_sumsq(rows, None, norm, y),
        "min_gru_scan": lambda: ops.min_gru_scan(*gru),
        "workspace": lambda: ops.Workspace(DEV).get("room", (1 << 20,), torch.float32).zero_(),
    }


def bits(got):
    return [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (got if isinstance(got, tuple) else (got,))]


NAMES = ["gemm", "gemm float32", "gemm into out", "gemm with a tile", "gemm in parts", "gemm_gated", "quantize", "quantize into out", "add_rmsnorm",
         "add_rmsnorm into out", "gated", "gated gelu", "add_weight_sumsq", "min_gru_scan", "workspace"]


@pytest.mark.parametrize("name", NAMES)
def test_room_is_of_the_launch_s_stream(name):
    from purhie_b200.csrc import ops
    call = calls()[name]
    want = [t.clone() for t in bits(call())]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    pool = torch.cuda.MemPool()
    with torch.cuda.stream(side), ops.on_current_stream():
        with torch.cuda.stream(torch.cuda.default_stream()), torch.cuda.use_mem_pool(pool):
            got = call()
    torch.cuda.synchronize()
    segments = pool.snapshot()
    assert segments and all(s["stream"] == side.cuda_stream for s in segments)
    if name != "min_gru_scan":                               # (its state has moved on)
        assert all(torch.equal(a, b) for a, b in zip(bits(got), want))


def test_parts_are_not_handed_out_while_they_are_added_up():
    """The scope's stream is busy, the current one fills new tensors of the parts' size as soon as a call has returned."""
    from purhie_b200.csrc import fp8, ops
    M, N, K = 24, 4096, 2304
    x, xs, w, ws = operands(M, N, K, 3)
    _, parts = fp8.plan(M, N, K)
    want = fp8.gemm(x, xs, w, ws).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side), ops.on_current_stream():
            torch.cuda._sleep(200_000)
            with torch.cuda.stream(torch.cuda.default_stream()):
                got = [fp8.gemm(x, xs, w, ws) for _ in range(3)]
                junk = [torch.full((parts, M, N), float("nan"), device=DEV) for _ in range(6)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got) and all(torch.isnan(j).all() for j in junk)
        del got, junk
