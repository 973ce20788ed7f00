"""Models whose matrices are held in 8 bits (option "gemm": "fp8"), through the engine's entry points."""
import math

import numpy as np
import pytest
import torch
from safetensors.torch import save_file

from plain import qwen3_plain as P
from helpers import make_model, random_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"

# widths that end inside a block of 128 and such that fill several; three requests' worth of grouped heads
SMALL = dict(architectures=["Qwen3ForCausalLM"], num_hidden_layers=3, hidden_size=272, intermediate_size=656, num_attention_heads=4,
             num_key_value_heads=2, head_dim=64, vocab_size=512, max_position_embeddings=512, rope_theta=1e6, rms_norm_eps=1e-6,
             tie_word_embeddings=False)
INIT = dict(seed=11, std=0.06, scale_low=0.8, scale_high=1.2, page_size=16)


def to_eight_bits(x, rows):
    """x (float64) as the values its e4m3 form stands for: a scale for each `rows` x 128."""
    t, k = x.shape
    p = x.new_zeros(-(-t // rows) * rows, -(-k // 128) * 128)
    p[:t, :k] = x
    b = p.view(-1, rows, p.shape[1] // 128, 128)
    s = b.abs().amax(dim=(1, 3), keepdim=True).clamp(min=448.0 * 2.0 ** -126) / 448.0
    v = b / s
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return ((torch.round(v / step) * step).clamp(-448, 448) * s).reshape(p.shape)[:t, :k]


def plain_eight_bit(cfg, w, tokens):
    """The forward pass with every product of a layer in 8 bits, in float64: weights in the layouts that the parts multiply by
    ([q | k | v] in one matrix, gate and up rows in turn)."""
    eps, positions = cfg["rms_norm_eps"], list(range(len(tokens)))
    HQ, HKV, D, E = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], cfg["hidden_size"]
    x = P.embedding(w["model.embed_tokens.weight"], tokens)
    T = len(tokens)
    for l in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{l}."
        qkv = to_eight_bits(torch.cat([w[p + f"self_attn.{n}_proj.weight"] for n in "qkv"]), 128)
        h = to_eight_bits(P.rmsnorm(x, w[p + "input_layernorm.weight"], eps), 1) @ qkv.T
        q, k, v = h.split([HQ * D, HKV * D, HKV * D], 1)
        q = P.rope_rotate_half(P.rmsnorm(q.reshape(T, HQ, D), w[p + "self_attn.q_norm.weight"], eps), positions, cfg["rope_theta"], D)
        k = P.rope_rotate_half(P.rmsnorm(k.reshape(T, HKV, D), w[p + "self_attn.k_norm.weight"], eps), positions, cfg["rope_theta"], D)
        o = P.attention(q, k, v.reshape(T, HKV, D), 1.0 / math.sqrt(D)).reshape(T, HQ * D)
        x = x + to_eight_bits(o, 1) @ to_eight_bits(w[p + "self_attn.o_proj.weight"], 128).T
        gu = torch.stack([w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"]], 1).reshape(-1, E)
        y = to_eight_bits(P.rmsnorm(x, w[p + "post_attention_layernorm.weight"], eps), 1) @ to_eight_bits(gu, 128).T
        g, u = y[:, 0::2], y[:, 1::2]
        x = x + to_eight_bits(g / (1.0 + torch.exp(-g)) * u, 1) @ to_eight_bits(w[p + "mlp.down_proj.weight"], 128).T
    return P.rmsnorm(x, w["model.norm.weight"], eps) @ w["lm_head.weight"].T


def rms_err(got, want):
    got, want = torch.as_tensor(np.asarray(got)).double(), want.double()
    return ((got - want).norm() / want.norm()).item()


@pytest.fixture(scope="module")
def small(tmp_path_factory):
    d = tmp_path_factory.mktemp("small8")
    make_model(d, SMALL, INIT, "bfloat16")
    cfg, w = P.read_model(str(d))
    tokens = random_tokens(230, SMALL["vocab_size"], 5)
    return str(d), tokens, plain_eight_bit(cfg, w, tokens), P.forward(cfg, w, tokens)


def load(folder, **options):
    from purhie_b200.api import load_model
    return load_model(folder, "bfloat16", options)


def test_logits_are_those_of_eight_bits(small):
    """A prompt in portions of different sizes (each kind of tile), then single tokens from the captured graph.  The engine's
    numbers between two roundings to 8 bits carry its bfloat16 roundings, so now and then a value falls to the other side: its
    error is then one step where the rounding itself is off by up to half a one.  All values doing that at once would be twice
    what the roundings move the logits by."""
    folder, tokens, eight, full = small
    moved = rms_err(eight, full)
    assert 0.005 < moved < 0.2                                       # 8 bits are seen in the logits, and no more than that
    for portions in ([1, 7, 40, 80, 2], [100, 30], [130]):
        model = load(folder, gemm="fp8")
        model.kv_cache_init(512, max_sequences=2)
        got, at = [], 0
        for n in portions:
            got.append(model.prefill_logits(tokens[at:at + n]))
            at += n
        assert rms_err(np.concatenate(got), eight[:at]) < 2 * moved, portions
        rows = []
        for t in tokens[at:at + 60]:
            model.decode_token(t)
            rows.append(model.get_logits())
        assert rms_err(np.stack(rows), eight[at:at + 60]) < 2 * moved, portions
        model.synchronize()
        model.free()


def test_weights_take_half_the_memory(small):
    folder = small[0]
    sizes = {}
    for gemm in ("auto", "fp8"):
        model = load(folder, gemm=gemm)
        model.kv_cache_init(128)
        sizes[gemm] = model.engine_info()["weight_bytes"]
        model.free()
    L, E, F, A = 3, 272, 656, 4 * 64 + 2 * 2 * 64
    matrices = L * (A * E + E * 4 * 64 + 3 * E * F)
    scales = 4 * L * (4 * 3 + 3 * 2 + 11 * 3 + 3 * 6)
    assert sizes["auto"] - sizes["fp8"] == matrices - scales


def test_every_way_of_generating(small):
    """Streams beside each other, the request queue, and one sequence: greedy tokens from the same logits (a near tie may
    fall either way, so the first tokens are compared with the formula's)."""
    folder, tokens, eight, _ = small
    model = load(folder, gemm="fp8")
    model.kv_cache_init(256, max_sequences=4)
    best = int(eight[99].argmax())
    margin = (eight[99].max() - eight[99].topk(2).values[1]).item() / eight[99].abs().max().item()
    out = model.generate([tokens[:100], tokens[:33], tokens[:100]], max_new_tokens=12)
    assert [len(o) for o in out] == [12, 12, 12] and out[0] == out[2]
    if margin > 0.05:
        assert out[0][0] == best
    again = model.generate([tokens[:100]], max_new_tokens=12)
    assert again[0][0] == out[0][0]
    model.synchronize()
    model.free()


def test_refusals(small):
    from purhie_b200.api import load_model
    from purhie_b200.native import InferenceError
    with pytest.raises(InferenceError, match="bfloat16 model"):
        load_model(small[0], "float32", {"gemm": "fp8"})


def feed_forward_probe(tmp_path, E, F, activation, options):
    from purhie_b200.csrc.build import build_library
    from purhie_b200.parts import PartProbe
    build_library("fp8")
    names = {k: k for k in ("gate_proj", "up_proj", "down_proj")}
    params = {"hidden_size": E, "intermediate_size": F, "names": names}
    if activation:
        params["activation"] = activation
    probe = PartProbe("feed_forward", "swiglu", params, "bfloat16", options)
    g = torch.Generator().manual_seed(E)
    w = {"gate_proj": torch.randn(F, E, generator=g) * E ** -0.5, "up_proj": torch.randn(F, E, generator=g) * E ** -0.5,
         "down_proj": torch.randn(E, F, generator=g) * F ** -0.5}
    w = {k: v.to(torch.bfloat16) for k, v in w.items()}
    d = tmp_path / "w"
    d.mkdir(exist_ok=True)
    save_file(w, str(d / "model.safetensors"))
    probe.bind_folder(str(d))
    return probe, {k: v.to(DEV) for k, v in w.items()}


@pytest.mark.parametrize("T,F", [(1, 656), (5, 656), (40, 656), (300, 656), (700, 656), (9, 2048), (600, 2048), (1500, 2048)])
@pytest.mark.parametrize("activation,gate", [(None, None), ({"kind": "clamped_swish", "alpha": 1.7, "limit": 3.0, "shift": 1.0}, (1.7, 3.0, 1.0)),
                                             ({"kind": "gelu_tanh"}, "gelu_tanh")])
def test_feed_forward_part_is_the_faces_one_after_the_other(T, F, activation, gate, tmp_path):
    """The part launches what the faces launch: the same bits."""
    from purhie_b200.csrc import fp8
    E = 272
    probe, w = feed_forward_probe(tmp_path, E, F, activation, {"gemm": "fp8"})
    x = torch.randn(T, E, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    got = torch.from_numpy(probe.feed_forward(x.float().numpy()))
    gu, gus = fp8.quantize(torch.stack([w["gate_proj"], w["up_proj"]], 1).reshape(-1, E).contiguous(), block_rows=128)
    dn, dns = fp8.quantize(w["down_proj"], block_rows=128)
    q, s = fp8.quantize(x.to(DEV))

    def product(q, s, w, ws, dtype):
        # as the parts ask for it: the parts of K, where there are several, go to whoever reads them
        tile, splits = fp8.plan(q.shape[0], w.shape[0], w.shape[1], whole=False)
        return fp8.gemm(q, s, w, ws, tile=tile, splits=splits, out_dtype=dtype), splits
    if F % 128 == 0 and fp8.plan(T, 2 * F, E) == (256, 1):
        q2, s2 = fp8.gemm_gated(q, s, gu, gus, gate=gate)
    else:
        y, n = product(q, s, gu, gus, torch.bfloat16)
        q2, s2 = fp8.gated(y, splits=n, gate=gate)
    out, n = product(q2, s2, dn, dns, torch.float32)
    if n > 1:
        out = out.double().sum(0).float()                            # the probe adds the parts up in double precision
    same = torch.equal(got, out.cpu())
    assert same


def test_weights_are_whole_before_they_are_brought_to_8_bits(tmp_path):
    """A matrix of a little more than 1 MiB: a copy from a file's mapping may return before its end is on the device."""
    E, F = 272, 2048
    x = torch.randn(9, E, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).float().numpy()
    got = []
    for i in range(8):
        (tmp_path / str(i)).mkdir()
        probe, _ = feed_forward_probe(tmp_path / str(i), E, F, None, {"gemm": "fp8"})
        got.append(probe.feed_forward(x))
    plain, _ = feed_forward_probe(tmp_path, E, F, None, {"gemm": "auto"})
    want = plain.feed_forward(x)
    for g in got:
        assert np.array_equal(g, got[0])
        # the last block of features, which the end of the matrix holds, is as near as all of them
        assert np.linalg.norm((g - want)[:, 256:]) < 0.1 * np.linalg.norm(want[:, 256:])


@pytest.mark.parametrize("options", [{"gemm": "fp8"}, {"gemm": "auto"}])
def test_a_matrix_under_one_name_for_two_products(options, tmp_path):
    """What the first product does with the weight when it is bound leaves the second one its own."""
    from purhie_b200.csrc.build import build_library
    from purhie_b200.parts import PartProbe
    build_library("fp8")
    E = 272
    w = (torch.randn(E, E, generator=torch.Generator().manual_seed(5)) * E ** -0.5).to(torch.bfloat16)
    got = []
    for i, names in enumerate(({"up_proj": "w", "down_proj": "w"}, {"up_proj": "w", "down_proj": "v"})):
        d = tmp_path / str(i)
        d.mkdir()
        save_file({n: w.clone() for n in set(names.values())}, str(d / "model.safetensors"))
        probe = PartProbe("feed_forward", "mlp", {"hidden_size": E, "intermediate_size": E, "activation": "silu", "names": names}, "bfloat16", options)
        probe.bind_folder(str(d))
        got.append(probe.feed_forward(torch.randn(9, E, generator=torch.Generator().manual_seed(6)).numpy()))
    assert np.isfinite(got[0]).all() and np.abs(got[0]).max() > 0 and np.array_equal(got[0], got[1])


def test_matrices_that_do_not_fit_stay_as_they_are(tmp_path):
    """Rows of a number of values that is no multiple of 16 stay in bfloat16: the same bits as without the option."""
    E, F = 264, 656
    x = torch.randn(9, E, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).float().numpy()
    eight, _ = feed_forward_probe(tmp_path, E, F, None, {"gemm": "fp8"})
    plain, _ = feed_forward_probe(tmp_path, E, F, None, {"gemm": "auto"})
    a, b = eight.feed_forward(x), plain.feed_forward(x)
    # the first product is the same, the second is in 8 bits
    assert not np.array_equal(a, b) and np.linalg.norm(a - b) < 0.1 * np.linalg.norm(b)
    narrow, _ = feed_forward_probe(tmp_path, 264, 648, None, {"gemm": "fp8"})
    same, _ = feed_forward_probe(tmp_path, 264, 648, None, {"gemm": "auto"})
    assert np.array_equal(narrow.feed_forward(x), same.feed_forward(x))


@pytest.mark.parametrize("design", ["bozosun", "sizizen", "zerusun", "vokepel", "noditar", "defapel"])
@pytest.mark.parametrize("which", ["CONFIG_A", "CONFIG_C"])
def test_every_design_loads_and_answers(design, which):
    """What the other designs' parts do with the option: attention and feed-forwards in 8 bits, the rest as it is.  Logits are near
    those in bfloat16 (a scale or a layout that is wrong would move them by their own size; a token that takes another expert moves
    its own row, so the middle row is looked at)."""
    import importlib
    from purhie_b200.api import load_model_random
    config = getattr(importlib.import_module(f"{design}_helpers"), which)
    tokens = random_tokens(80, config["vocab"], 3)
    got = {}
    for gemm in ("auto", "fp8"):
        model = load_model_random(config, 5, "bfloat16", std=0.1, options={"gemm": gemm})
        model.kv_cache_init(96, max_sequences=2)
        rows = [model.prefill_logits(tokens[:50]), model.prefill_logits(tokens[50:70])]
        for t in tokens[70:]:
            model.decode_token(t)
            rows.append(model.get_logits()[None])
        model.synchronize()
        model.free()
        got[gemm] = np.concatenate(rows).astype(np.float64)
    assert np.isfinite(got["fp8"]).all()
    far = np.linalg.norm(got["fp8"] - got["auto"], axis=1) / np.linalg.norm(got["auto"], axis=1)
    assert np.median(far) < 0.3, far
