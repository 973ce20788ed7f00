"""The parts of a layer whose matrices are held in 8 bits, bit for bit beside the faces.

A part's first product is followed by kernels of its own (norms, rotation, attention, an activation), so it is fed with numbers
whose product is the same in 8 bits and in bfloat16: every block holds small whole numbers and one value of 448, times a power of
two that differs from block to block.  Its scale is that power of two, nothing is rounded, and a scale of another block would double or
halve what it multiplies.  The sums are whole numbers of at most 256, which bfloat16 holds too.  With the identity as its second matrix the
same part in bfloat16 then gives what goes into the second product, and the faces say what that product makes of it in 8 bits.
"""
import numpy as np
import pytest
import torch
from safetensors.torch import save_file

pytestmark = pytest.mark.gpu
DEV = "cuda"


def exponents(rows, K, each, g):
    """0 or 1 for each block of `each` x 128, spread over a matrix."""
    e = torch.randint(0, 2, (-(-rows // each), -(-K // 128)), generator=g)
    return e.repeat_interleave(each, 0)[:rows].repeat_interleave(128, 1)[:, :K]


def last_columns(K, back):
    """The column `back` in front of each block's end."""
    return [min(b + 128, K) - 1 - back for b in range(0, K, 128)]


def exact_rows(T, K, g):
    """Whole numbers of at most 4, with a 448 in each block's last column, where no weight is; none in the column in front of it."""
    x = torch.randint(-4, 5, (T, K), generator=g).float()
    x[:, last_columns(K, 0)] = 448.0
    x[:, last_columns(K, 1)] = 0.0
    return x * 2.0 ** exponents(T, K, 1, g)


def exact_weight(N, K, g):
    """Eight numbers of at most 2 a row (8 * 8 * 4 = 256 with the powers of two), with a 448 in each block, where no row of x has anything."""
    w = torch.zeros(N, K)
    free = torch.tensor([k for k in range(K) if k not in last_columns(K, 0) + last_columns(K, 1)])
    for n in range(N):
        at = free[torch.randperm(len(free), generator=g)[:8]]
        w[n, at] = torch.tensor([-2.0, -1.0, 1.0, 2.0])[torch.randint(0, 4, (8,), generator=g)]
    for c in last_columns(K, 1):
        w[::128, c] = 448.0
    return w * 2.0 ** exponents(N, K, 128, g)


def part(tmp_path, name, family, kind, params, options, weights):
    from purhie_b200.csrc.build import build_library
    from purhie_b200.parts import PartProbe
    build_library("fp8")
    probe = PartProbe(family, kind, params, "bfloat16", options)
    roles = {s["name"]: s["role"] for s in probe.tensor_specs()}
    d = tmp_path / name
    d.mkdir()
    save_file({n: t.to(torch.bfloat16 if roles[n] == "matrix" else torch.float32).contiguous() for n, t in weights.items()}, str(d / "model.safetensors"))
    probe.bind_folder(str(d))
    return probe


def product_of(rows, weight):
    """What a part's product gives for bfloat16 rows: brought to 8 bits, multiplied in the parts that the plan says; the probe adds the
    parts up in double precision."""
    from purhie_b200.csrc import fp8
    q, s = fp8.quantize(rows.to(DEV, torch.bfloat16))
    w, ws = fp8.quantize(weight.to(DEV, torch.bfloat16), block_rows=128)
    tile, splits = fp8.plan(q.shape[0], w.shape[0], w.shape[1], whole=False)
    y = fp8.gemm(q, s, w, ws, tile=tile, splits=splits, out_dtype=torch.float32)
    return (y.double().sum(0).float() if splits > 1 else y).cpu().numpy()


STEPS = [
    [[(0, 1)]],                                                            # one token
    [[(r, 1) for r in range(8)], [(r, 1) for r in range(8)]],              # eight, twice
    [[(0, 37)], [(0, 1), (1, 50), (2, 1)]],                                # portions beside tokens
    [[(0, 96), (3, 4)], [(3, 1), (0, 1)]],
    [[(0, 200), (1, 100)], [(1, 399), (0, 1), (2, 300)]],                  # tiles of 256 rows
]
NAMES = {k: k for k in ("q_proj", "k_proj", "v_proj", "o_proj", "q_norm", "k_norm", "gate_proj")}


def attention_pair(tmp_path, kind, gate, HQ, HKV, D):
    """The part in bfloat16 with the identity as its output matrix, the part in 8 bits, and that one's output matrix."""
    E = HQ * D
    g = torch.Generator().manual_seed(HQ + D)
    names = {k: v for k, v in NAMES.items() if gate or k != "gate_proj"}
    params = {"hidden_size": E, "num_heads": HQ, "num_kv_heads": HKV, "head_dim": D, "names": names}
    if kind == "attention":
        params.update(qk_norm_eps=1e-5, position={"kind": "rope_neox", "params": {"theta": 5e4, "n_rot": D, "max_position": 1024}})
    else:
        params.update(joint_norm_eps=1e-5)
    widths = [HQ * D, HKV * D, HKV * D] + ([HQ * D] if gate else [])
    first = exact_weight(sum(widths), E, g).split(widths)
    w = dict(zip(["q_proj", "k_proj", "v_proj", "gate_proj"], first))
    heads = (HQ, HKV) if kind == "talking_attention" else (1, 1)           # (its norms span all heads)
    w.update(q_norm=1 + 0.3 * torch.randn(heads[0] * D, generator=g), k_norm=1 + 0.3 * torch.randn(heads[1] * D, generator=g))
    o = (torch.randn(E, E, generator=g) * E ** -0.5).to(torch.bfloat16)
    plain = part(tmp_path, "plain", "mixer", kind, params, {"gemm": "auto"}, dict(w, o_proj=torch.eye(E)))
    eight = part(tmp_path, "eight", "mixer", kind, params, {"gemm": "fp8"}, dict(w, o_proj=o))
    return plain, eight, o, E, g


@pytest.mark.parametrize("steps", STEPS, ids=["one", "eight", "portions", "hundred", "many"])
@pytest.mark.parametrize("kind,gate,HQ,HKV,D", [("attention", False, 5, 1, 64), ("attention", False, 4, 2, 80), ("attention", True, 3, 1, 128),
                                                ("talking_attention", False, 5, 1, 64), ("talking_attention", True, 4, 2, 80)])
def test_attention_s_products_are_the_faces(kind, gate, HQ, HKV, D, steps, tmp_path):
    """Query, key, value (and gate) products through the attention kernels, then the output product; rows that come in bfloat16 and in 8
    bits; and a layer that reads another one's cache, whose product is the first rows of the same matrix (a width that ends inside a
    block)."""
    plain, eight, o, E, g = attention_pair(tmp_path, kind, gate, HQ, HKV, D)
    for probe in (plain, eight):
        probe.mixer_cache(16, 256, max_requests=24)
        for r in range(24):
            probe.add_request(r)
    reads = kind == "attention" and not gate
    for step in steps:
        x = exact_rows(sum(n for _, n in step), E, g).numpy()
        rows = torch.from_numpy(plain.mixer_step(step, x))
        assert torch.equal(rows, rows.to(torch.bfloat16).float()) and rows.abs().max() > 0
        want = product_of(rows, o)
        assert np.array_equal(eight.mixer_step(step, x), want)
        # the same step for other requests, its rows in 8 bits, and read by a second layer
        moved = [(8 + r, n) for r, n in step]
        assert np.array_equal(eight.mixer_step(moved, x, eight_bit=True), want)
        if reads:
            again = [(16 + r, n) for r, n in step]
            assert np.array_equal(eight.mixer_step(again, x, reads_only=True), want)


@pytest.mark.parametrize("T", [1, 40, 300, 700])
def test_ungated_feed_forward_is_the_faces(T, tmp_path):
    E = 272
    g = torch.Generator().manual_seed(T)
    params = {"hidden_size": E, "intermediate_size": E, "activation": "silu", "names": {"up_proj": "u", "down_proj": "d"}}
    up, down = exact_weight(E, E, g), (torch.randn(E, E, generator=g) * E ** -0.5).to(torch.bfloat16)
    plain = part(tmp_path, "plain", "feed_forward", "mlp", params, {"gemm": "auto"}, {"u": up, "d": torch.eye(E)})
    eight = part(tmp_path, "eight", "feed_forward", "mlp", params, {"gemm": "fp8"}, {"u": up, "d": down})
    x = exact_rows(T, E, g).numpy()
    want = product_of(torch.from_numpy(plain.feed_forward(x)), down)
    assert np.array_equal(eight.feed_forward(x), want) and np.array_equal(eight.feed_forward(x, eight_bit=True), want)


@pytest.mark.parametrize("T,F", [(1, 656), (40, 656), (300, 656), (9, 2048), (1500, 2048)])
def test_gated_feed_forward_takes_rows_in_8_bits(T, F, tmp_path):
    E = 272
    g = torch.Generator().manual_seed(T)
    w = {"gate_proj": torch.randn(F, E, generator=g) * E ** -0.5, "up_proj": torch.randn(F, E, generator=g) * E ** -0.5, "down_proj": torch.randn(E, F, generator=g) * F ** -0.5}
    probe = part(tmp_path, "eight", "feed_forward", "swiglu", {"hidden_size": E, "intermediate_size": F, "names": {k: k for k in w}}, {"gemm": "fp8"}, w)
    x = torch.randn(T, E, generator=g).numpy()
    assert np.array_equal(probe.feed_forward(x), probe.feed_forward(x, eight_bit=True))


@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("add,parts", [(None, 1), ("float32", 1), ("bfloat16", 1), ("float32", 5)])
@pytest.mark.parametrize("T,E", [(1, 64), (7, 272), (150, 1000), (3, 4104), (2, 32768)])
def test_norm_in_8_bits_is_the_face(T, E, add, parts, offset, tmp_path):
    from purhie_b200.csrc import fp8
    g = torch.Generator().manual_seed(E)
    weight = 1 - offset + 0.3 * torch.randn(E, generator=g)
    norm = part(tmp_path, "norm", "norm", "rmsnorm", {"size": E, "eps": 1e-5, "weight_offset": offset, "names": {"weight": "w"}}, {"gemm": "fp8"}, {"w": weight})
    x = torch.randn(T, E, generator=g) * 3
    a = None if add is None else torch.randn(parts, T, E, generator=g).to(getattr(torch, add))
    out_x, q, scales = norm.norm_eight_bit(x.numpy(), None if a is None else a.float().numpy(), add or "float32")
    kept = x.to(DEV)
    want_q, want_s = fp8.add_rmsnorm(kept, None if a is None else a.to(DEV), (weight + offset).to(DEV), 1e-5, add_splits=parts)
    assert np.array_equal(out_x, kept.cpu().numpy())
    assert np.array_equal(q, want_q.view(torch.uint8).cpu().numpy()) and np.array_equal(scales, want_s.cpu().numpy())


@pytest.mark.parametrize("T", [1, 20])
def test_a_layer_s_parts_hand_rows_on_in_8_bits(T):
    """The launches of a step: each layer's two norms and its activation give the next product's rows, and the attention's output alone
    goes through the quantizer; the norm in front of the output matrix is the one left in bfloat16."""
    from purhie_b200 import native
    from purhie_b200.engine import Engine, StepEntry
    config = dict(architectures=["Qwen3ForCausalLM"], num_hidden_layers=3, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                  vocab_size=512, max_position_embeddings=512, rope_theta=1e6, rms_norm_eps=1e-6, tie_word_embeddings=False)
    eng = Engine.from_random(config, 3, dtype="bfloat16", max_tokens=1024, max_requests=1, options={"gemm": "fp8"})
    eng.add_request(0)
    eng.step([StepEntry(0, list(range(20)), [])])
    native.lib().qe_profile_enable(1)
    try:
        native.profile_report()
        eng.step([StepEntry(0, list(range(T)), [T - 1])])
        report = native.profile_report()
    finally:
        native.lib().qe_profile_enable(0)
    eng.close()
    calls = {k: v["calls"] for k, v in report.items()}
    assert (calls["quantize"], calls["gated"], calls["add_rmsnorm"]) == (3, 3, 7), calls
    assert "swiglu" not in calls and "add_weight_sumsq" not in calls, calls
