"""fp8 checkpoints (e4m3 projections, a scale for each 128 x 128) through the model classes.  CPU: codes, the files' checks.  GPU (-m gpu): against the oracle.

What may differ from the oracle: f32 sums in another order, 1e-6 of a row (one token's pass), and attention in split precision, 1e-5 at most (prompts).  Where that moves
an activation across the border of two codes its code differs by a step: a share 2 x 1e-5 / 2^-4 = 3e-4 of a prompt's elements, 3e-5 of one token's.
  No code differs: 1e-4 of the logits.  A pass of one token through three layers of width 256 forms 3 x (4 x 256 + 512) codes, 0.15 of them differ, six passes of seven have none; half
  of sixteen are asked for.  The same of short prompts through one layer (2 and 17 rows).
  Longer prompts: the norm of the table's bf16 rows gives quotients of short numbers, which fall on the border of two codes exactly every 2^8 / 2^4 x 2^10 = 16 000 elements or so
  (8 bits against the border's 4, and the product of norm weight and 1 / rms takes a tie off in all but one of 2^10), one row of 64: the first q, k and v are asked to agree to
  1e-5 in nine rows of ten, and what follows, which reads all keys, to the bound below.
  Some differ: a step is up to 2^-3 of its element, and moves the row by up to 1e-2 of itself; that is 2^-4 of an element and more, so from there on the codes of the two sides round
  apart, each off by its own rounding.  Two independent roundings lie sqrt(2) times as far from each other as one from the unrounded activations, which the oracle
  computes too (`gap`); with the scatter of a largest difference over the vocabulary from pass to pass, a factor 2: 3 times the largest gap.  (First set at 0.01 and 0.061, as
  if one code's difference stayed alone.)"""
import ctypes as C
import json
import struct

import numpy as np
import pytest

import crane_b200
from conftest import rel_err
from crane_b200 import CraneB200Error, synth

TINY = synth.fp8_config(synth.TINY_QWEN3)


def test_codes_are_e4m3():
    import torch
    v = synth.e4m3_values()
    assert np.array_equal(torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy(), v)
    x = np.concatenate([v, -v, (v[1:] + v[:-1]) / 2, np.random.default_rng(0).standard_normal(4096).astype(np.float32) * 40]).astype(np.float32)
    assert np.array_equal(synth.e4m3_encode(x), torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert np.array_equal(synth.e4m3_decode(synth.e4m3_encode(v)), v)


def write_safetensors(path, tensors):
    kinds = {np.dtype(np.uint8): "F8_E4M3", np.dtype(np.uint16): "BF16", np.dtype(np.float32): "F32"}
    head, data = {}, b""
    for name, a in tensors.items():
        head[name] = {"dtype": kinds[a.dtype], "shape": list(a.shape), "data_offsets": [len(data), len(data) + a.nbytes]}
        data += a.tobytes()
    h = json.dumps(head).encode()
    path.write_bytes(struct.pack("<Q", len(h)) + h + data)


def model(cfg=TINY, tensors=None, **opts):
    m = crane_b200.model_class(cfg)(cfg, device=0, **{"max_seq_len": 256, **opts})
    m.load_checkpoint((tensors or dict(synth.fp8_checkpoint(cfg))).items())
    return m


def gap_of(w, cfg, passes):
    """The largest difference that rounding the activations makes to the logits of some passes: lists of (ids, start)."""
    from oracle.fp8 import Fp8Oracle
    out = []
    for p in passes:
        a, b = Fp8Oracle(cfg, w), Fp8Oracle(cfg, w, plain=True)
        out += [rel_err(b.forward(ids, at).numpy(), a.forward(ids, at).numpy()) for ids, at in p]
    return max(out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 70, 200])
def test_prompt_and_tokens_against_the_oracle(rows):
    from oracle.fp8 import Fp8Oracle
    w = dict(synth.fp8_checkpoint(TINY))
    orc = Fp8Oracle(TINY, w)
    m = model(tensors=w)
    ids = synth.synth_token_ids(rows, TINY["vocab_size"], "fp8")
    ref = orc.forward(ids, 0).numpy()
    errs, passes = [rel_err(m.forward_step(ids, 0), ref)], [(ids, 0)]
    for i in range(6):
        tok = int(ref.argmax())
        passes.append(([tok], rows + i))
        ref = orc.forward([tok], rows + i).numpy()
        errs.append(rel_err(m.forward_step([tok], rows + i), ref))
    gap = gap_of(w, TINY, [passes])
    print(f"fp8 {rows} rows: rel {max(errs):.2e}, rounding the activations {gap:.1e}")
    assert max(errs) < 3 * gap
    m.close()


@pytest.mark.gpu
def test_single_tokens_against_the_oracle():
    from oracle.fp8 import Fp8Oracle
    w = dict(synth.fp8_checkpoint(TINY))
    orc, m = Fp8Oracle(TINY, w), model(tensors=w)
    errs, toks = [], [int(t) for t in synth.synth_token_ids(16, TINY["vocab_size"], "fp8one")]
    for t in toks:
        orc.clear_kv_cache(), m.clear_kv_cache()
        errs.append(rel_err(m.forward_step([t], 0), orc.forward([t], 0).numpy()))
    print("fp8 single tokens:", " ".join(f"{e:.1e}" for e in errs))
    assert sum(e < 1e-4 for e in errs) >= 8 and max(errs) < 3 * gap_of(w, TINY, [[([t], 0)] for t in toks])
    m.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 17, 60, 90, 130, 250])
def test_prompts_through_one_layer_against_the_oracle(rows):
    """Lengths on every route of the linears (few rows, tiles of rows, pairs)."""
    from oracle.fp8 import Fp8Oracle
    cfg = dict(TINY, num_hidden_layers=1)
    w = dict(synth.fp8_checkpoint(cfg))
    m, prompts = model(cfg, tensors=w, max_seq_len=512), [synth.synth_token_ids(rows, cfg["vocab_size"], f"fp8p{i}") for i in range(8)]
    m.lib.crane_b200_debug_peek.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_size_t]
    seen = {}

    class Recording(Fp8Oracle):
        def _linear(self, name, x, w=None):
            seen[name.split(".")[-2]] = y = super()._linear(name, x, w)
            return y
    errs, near = [], []
    for ids in prompts:
        m.clear_kv_cache()
        errs.append(rel_err(m.forward_step(ids, 0), Recording(cfg, w).forward(ids, 0).numpy()))
        ref = np.concatenate([seen[n].numpy() for n in ("q_proj", "k_proj", "v_proj")], 1)
        qkv = np.empty_like(ref)
        m._ck(m.lib.crane_b200_debug_peek(m.h, 1, qkv.ctypes.data, qkv.size))
        near.append((np.abs(qkv - ref).max(1) < 1e-5 * np.abs(ref).max()).mean())
    print(f"fp8 prompts of {rows}, one layer:", " ".join(f"{e:.1e}" for e in errs), "rows of q, k, v alike:", " ".join(f"{n:.2f}" for n in near))
    assert max(errs) < 3 * gap_of(w, cfg, [[(ids, 0)] for ids in prompts])
    assert np.mean(near) >= 0.9 and (rows > 17 or sum(e < 1e-4 for e in errs) >= 4)
    m.close()


@pytest.mark.gpu
def test_decode_batches_forks_and_greedy_loops_agree_with_single_steps():
    """Rounds of 1, 2, 3 and 5 sequences, a fork, and the on-device loop: the logits of the same sequences step by step, as near as the oracle is held to."""
    w = dict(synth.fp8_checkpoint(TINY))
    m = model(tensors=w, max_batch=6)
    prompts = [synth.synth_token_ids(n, TINY["vocab_size"], f"fp8b{n}") for n in (5, 17, 33, 64, 100)]
    want = []
    for p in prompts:
        m.clear_kv_cache()
        first = m.forward_step(p, 0)
        want.append((int(first.argmax()), m.forward_step([int(first.argmax())], len(p))))
    gap = gap_of(w, TINY, [[(p, 0), ([t], len(p))] for p, (t, _) in zip(prompts, want)])
    for n in (1, 2, 3, 5):
        seqs, toks = [], []
        for p, (t, _) in list(zip(prompts, want))[:n]:
            s = m.seq_create()
            m.seq_select(s)
            m.forward_step(p, 0)
            seqs.append(s), toks.append(t)
        if n == 3:
            seqs.append(m.seq_fork(seqs[1])), toks.append(toks[1])
        _, logits = m.decode_batch(seqs, toks, 1, want_logits=True)
        for i, s in enumerate(seqs):
            assert rel_err(logits[i], want[1 if i == 3 and n == 3 else i][1]) < 3 * gap
            m.seq_free(s)
    m.seq_select(0)
    m.clear_kv_cache()
    assert len(m.generate(prompts[2], max_new_tokens=12)) == 12
    m.close()


@pytest.mark.gpu
def test_two_handles_on_two_streams_and_repeats():
    """Two handles in turn answer what each answers alone, bit for bit, from graphs and kernel by kernel."""
    w = dict(synth.fp8_checkpoint(TINY))
    ids = synth.synth_token_ids(40, TINY["vocab_size"], "fp8t")
    out = []
    for opts in ({}, {"graphs": False}, {"pdl": False}):
        a, b = model(tensors=w, **opts), model(tensors=w, **opts)
        la = [a.forward_step(ids, 0), b.forward_step(ids, 0)]
        la += [m.forward_step([int(ids[i])], 40 + i) for i in range(4) for m in (a, b)]
        for x, y in zip(la[0::2], la[1::2]):
            assert np.array_equal(x, y)
        out.append(la)
        a.close(), b.close()
    for x in out[1:]:
        for p, q in zip(out[0], x):
            assert np.array_equal(p, q)


@pytest.mark.gpu
def test_a_safetensors_file_and_the_vision_model(tmp_path):
    """The file reader takes F8_E4M3 tensors and bf16 scales; the VL model's text layers may be e4m3."""
    w = {n: (a if a.dtype == np.uint8 else synth.f32_to_bf16_bits(a)) for n, a in synth.fp8_checkpoint(TINY)}
    path = tmp_path / "model.safetensors"
    write_safetensors(path, w)
    m = crane_b200.Qwen3Model(TINY, device=0, max_seq_len=256)
    loaded, skipped = m.load_safetensors(str(path))
    m.finalize()
    assert (loaded, skipped) == (len(w), 0)
    ids = synth.synth_token_ids(20, TINY["vocab_size"], "fp8f")
    back = {n: (a if a.dtype == np.uint8 else synth.bf16_bits_to_f32(a)) for n, a in w.items()}
    other = model(tensors=back)
    assert np.array_equal(m.forward_step(ids, 0), other.forward_step(ids, 0))
    m.close(), other.close()
    cfg = synth.fp8_config(synth.TINY_QWEN3_VL)
    vl = model(cfg)
    assert np.isfinite(vl.forward_step(synth.synth_token_ids(9, synth.text_config(cfg)["vocab_size"], "fp8v"), 0)).all()
    vl.close()


@pytest.mark.gpu
def test_what_does_not_fit_is_refused():
    w = dict(synth.fp8_checkpoint(TINY))
    q = next(n for n in w if n.endswith("0.self_attn.q_proj.weight"))

    def refused(cfg, tensors, said):
        m = crane_b200.Qwen3Model(cfg, device=0, max_seq_len=256)
        with pytest.raises(CraneB200Error, match=said):
            m.load_checkpoint(tensors.items())
        m.close()
    refused(synth.TINY_QWEN3, w, "quantization_config")                                       # codes, but the config says nothing of them
    refused(TINY, {n: a for n, a in w.items() if n != q + "_scale_inv"}, "do not match")
    refused(TINY, {**w, q + "_scale_inv": w[q + "_scale_inv"][:, :1]}, "shape")
    refused(TINY, {**w, q: w[q][:128]}, "shape")
    mixed = dict(w, **{q: synth.e4m3_decode(w[q])})
    del mixed[q + "_scale_inv"]
    refused(TINY, mixed, "all seven")
    norm = next(n for n in w if n.endswith("norm.weight"))
    refused(TINY, {**w, norm: np.zeros(w[norm].shape, np.uint8)}, "e4m3")
    emb = next(n for n in w if n.endswith("embed_tokens.weight"))
    refused(TINY, {**w, emb: np.zeros(w[emb].shape, np.uint8)}, "e4m3")
    for change in ({"weight_block_size": [64, 64]}, {"activation_scheme": "static"}, {"fmt": "e5m2"}, {"weight_block_size": None}):
        cfg = dict(TINY, quantization_config={**TINY["quantization_config"], **change})
        with pytest.raises(CraneB200Error, match="quantization_config"):
            crane_b200.Qwen3Model(cfg, device=0, max_seq_len=256)
