"""The seven projections of an fp8 checkpoint's layer inside the model classes, each on what the device itself gave the one ahead of it.

A prompt through one layer leaves q, k and v, the attention's output and the layer's result on the device (crane_b200_debug_peek). The operators of crane_b200.fp8, which test_fp8.py holds
to 64 bits, take the same rows through the checkpoint's tensors: the model runs the same kernels on the same rows, so the results are equal bit for bit, at every length."""
import ctypes as C

import numpy as np
import pytest
import torch

import crane_b200
from crane_b200 import synth

F8 = torch.float8_e4m3fn


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def matrix(w, *names):
    """(codes, scales) of projections below one another."""
    by = {n.split("layers.0.")[1]: a for n, a in w.items() if "layers.0." in n and "visual" not in n}
    return (cuda(np.concatenate([by[n + ".weight"] for n in names])).view(F8), cuda(np.concatenate([by[n + ".weight_scale_inv"] for n in names])))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["dense", "vl"])
def test_projections_of_a_layer(kind):
    from crane_b200 import fp8
    if kind == "dense":
        cfg = synth.fp8_config(dict(synth.TINY_QWEN3_UNTIED, num_hidden_layers=1))
    else:
        cfg = synth.fp8_config(dict(synth.TINY_QWEN3_VL, text_config=dict(synth.TINY_QWEN3_VL["text_config"], num_hidden_layers=1),
                                    vision_config=dict(synth.TINY_QWEN3_VL["vision_config"], deepstack_visual_indexes=[0])))
    t = synth.text_config(cfg)
    H, I, eps = t["hidden_size"], t["intermediate_size"], t["rms_norm_eps"]
    qd, kvd = t["num_attention_heads"] * t["head_dim"], t["num_key_value_heads"] * t["head_dim"]
    w = dict(synth.fp8_checkpoint(cfg))
    m = crane_b200.model_class(cfg)(cfg, device=0, max_seq_len=1024)
    m.load_checkpoint(w.items())
    m.lib.crane_b200_debug_peek.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_size_t]

    def peek(which, *shape):
        out = np.empty(shape, np.float32)
        m._ck(m.lib.crane_b200_debug_peek(m.h, which, out.ctypes.data, out.size))
        return cuda(out)
    norm = lambda end: next(cuda(a.astype(np.float32)) for n, a in w.items() if n.endswith("layers.0." + end))      # noqa: E731
    embed = next(a for n, a in w.items() if n.endswith("embed_tokens.weight") and "visual" not in n)
    embed = synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(embed.astype(np.float32)))
    qkv_w, o_w = matrix(w, "self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), matrix(w, "self_attn.o_proj")
    gu_w, down_w = matrix(w, "mlp.gate_proj", "mlp.up_proj"), matrix(w, "mlp.down_proj")
    for rows in (2, 16, 17, 33, 60, 90, 130, 257, 700):
        ids = synth.synth_token_ids(rows, min(t["vocab_size"], 1000), f"fp8q{rows}")
        m.clear_kv_cache()
        m.forward_step(ids, 0)
        x0, qkv, attn, x = cuda(embed[np.asarray(ids)]), peek(1, rows, qd + 2 * kvd), peek(2, rows, qd), peek(0, rows, H)
        assert torch.equal(fp8.linear(*fp8.rms_norm(x0, norm("input_layernorm.weight"), eps), *qkv_w, dtype=torch.float32), qkv), rows
        x1 = fp8.linear(*fp8.quantize(attn), *o_w, add=x0, dtype=torch.float32)
        gu = fp8.linear(*fp8.rms_norm(x1, norm("post_attention_layernorm.weight"), eps), *gu_w, dtype=torch.float32)
        assert torch.equal(fp8.linear(*fp8.silu_mul(gu), *down_w, add=x1, dtype=torch.float32), x), rows
        assert torch.isfinite(x).all() and float(x.abs().max()) > 0 and gu.shape == (rows, 2 * I)
    fp8.status()
    m.close()
