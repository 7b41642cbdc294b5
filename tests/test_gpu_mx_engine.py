"""An engine with microscaled weights against a plain statement of its layers in float64.

The plain model rounds where the engine rounds: matrices to 4 bits, the rows that enter a product to 8, keys, values and the
attention's output to bfloat16.  What is left is where a value that the engine's bfloat16 attention moves in its last place (2^-9)
falls on the other side of an 8-bit rounding (a step of 2^-4 to 2^-3): one element in 32 or so, by a sixteenth, about one percent
of a row's size at each of four roundings a layer.  Five percent of the largest logit holds that for the few layers here."""
import numpy as np
import pytest
import torch

import mx_util
import plain_qwen3 as plain
from util import TINY, assert_close_logits, make_model, random_tokens

pytestmark = pytest.mark.gpu
RTOL = 5e-2
F64 = torch.float64


def held(x, bits):
    """The numbers that rows have in the format."""
    x = np.asarray(x.to(torch.float64))
    codes, scales = mx_util.quantize(x, bits)
    return torch.from_numpy(mx_util.numbers(codes, scales, bits)[:, : x.shape[1]])


def plain_logits(cfg, w, tokens):
    heads, kv, hd, eps = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], cfg["rms_norm_eps"]
    x = plain.plain_embedding(w["model.embed_tokens.weight"], torch.tensor(tokens))
    s = len(tokens)
    angles = plain.plain_rope_angles(torch.arange(s), hd, cfg["rope_theta"])
    types = cfg.get("layer_types") or ["full_attention"] * cfg["num_hidden_layers"]
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        m = {n: held(w[p + n + ".weight"], 4) for n in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj",
                                                         "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")}
        h = held(plain.plain_rmsnorm(x, w[p + "input_layernorm.weight"], eps), 8)
        q, k, v = ((h @ m[f"self_attn.{n}_proj"].T).view(s, -1, hd) for n in "qkv")
        q = plain.plain_rope_neox(plain.plain_rmsnorm(q, w[p + "self_attn.q_norm.weight"], eps), angles)
        k = plain.plain_rope_neox(plain.plain_rmsnorm(k, w[p + "self_attn.k_norm.weight"], eps), angles)
        k, v = (t.to(torch.bfloat16).to(F64) for t in (k, v))
        window = cfg["sliding_window"] if types[i] == "sliding_attention" else None
        o = plain.plain_attention(q, k, v, hd ** -0.5, window).reshape(s, heads * hd).to(torch.bfloat16)
        x = x + held(o, 8) @ m["self_attn.o_proj"].T
        h = held(plain.plain_rmsnorm(x, w[p + "post_attention_layernorm.weight"], eps), 8)
        inner = held(plain.plain_swiglu(h @ m["mlp.gate_proj"].T, h @ m["mlp.up_proj"].T), 8)
        x = x + inner @ m["mlp.down_proj"].T
    h = plain.plain_rmsnorm(x, w["model.norm.weight"], eps).to(torch.bfloat16).to(F64)
    head = w["model.embed_tokens.weight" if cfg["tie_word_embeddings"] else "lm_head.weight"]
    return h @ head.to(F64).T


@pytest.mark.parametrize("name, lengths", [("A", (1, 40)), ("C", (90,)), ("D", (150, 7)), ("E", (200, 33))])
def test_logits(tmp_path, name, lengths):
    from tinyinfer_b200 import Engine, StepEntry
    folder = make_model(tmp_path, name)
    cfg, weights = plain.load_folder(folder)
    engine = Engine(folder, weights="mxfp4", max_requests=len(lengths))
    entries, want = [], []
    for r, n in enumerate(lengths):
        tokens = random_tokens(TINY[name]["vocab_size"], n, seed=n)
        engine.add_request(r)
        entries.append(StepEntry(r, tokens, want=list(range(n))))
        want.append(plain_logits(TINY[name], weights, tokens))
    got = engine.step(entries)
    engine.ops.check_status()
    assert_close_logits(got, torch.cat(want), RTOL, f"{name}, whole prompts")
    # the same prompts token by token behind half a prompt
    for r, n in enumerate(lengths):
        engine.finish(r)
        engine.add_request(r)
        tokens, half, rows = entries[r].tokens, max(1, n // 2), []
        rows.append(engine.step([StepEntry(r, tokens[:half], want=list(range(half)))]).clone())
        for t in tokens[half:half + 6]:
            rows.append(engine.step([StepEntry(r, [t], want=[0])]).clone())
        rows = torch.cat(rows)
        assert_close_logits(rows, want[r][: rows.shape[0]], RTOL, f"{name}, portions")
    engine.ops.check_status()


def test_generation_with_graphs_is_that_without(tmp_path):
    from tinyinfer_b200 import LLM, SamplingParams
    folder = make_model(tmp_path, "E")
    prompts = [random_tokens(TINY["E"]["vocab_size"], n, seed=n) for n in (70, 5, 130)]
    outs = []
    for graphs in (False, True):
        llm = LLM(folder, weights="mxfp4", max_seq=256, max_num_seqs=4, max_batched_tokens=160, cuda_graph=graphs)
        outs.append([g.tokens for g in llm.generate(prompts, SamplingParams(max_tokens=12))])
        llm.engine.ops.check_status()
    assert outs[0] == outs[1] and all(len(t) == 12 for t in outs[0])


def test_weights_take_about_a_quarter_of_the_memory(tmp_path):
    from tinyinfer_b200 import Engine
    from tinyinfer_b200.kernels import MxRows
    cfg = dict(TINY["E"], hidden_size=512, intermediate_size=1536, num_hidden_layers=1)
    block = Engine(config=cfg, seed=1, weights="mxfp4", max_requests=1).model.blocks[0]
    for w in (block.mixer.w_qkv, block.mixer.w_o, block.ffn.w_gate_up, block.ffn.w_down):
        assert isinstance(w, MxRows) and w.settled and w.bits == 4
        assert w.codes.numel() + w.scales.numel() <= 0.27 * 2 * w.rows * w.cols
