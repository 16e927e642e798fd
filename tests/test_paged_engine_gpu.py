"""The inference engine over 8-bit pages: the fp32 model's logits, prompts in portions, captured steps, limits, the command line."""
import json
import os

import numpy as np
import pytest
import torch

from paged_oracle import Seq, attention

pytestmark = pytest.mark.gpu


def cfg_of(**over):
    from ghassan_b200.models.config import ModelConfig
    base = dict(vocab_size=512, hidden_size=256, num_layers=2, num_heads=4, num_kv_heads=2, intermediate_size=512, max_seq_len=512, use_moe=True, num_experts=4,
                moe_top_k=2, moe_expert_dim=128, moe_shared=True, use_qk_norm=True)
    base.update(over)
    c = ModelConfig(**base)
    c.validate()
    return c


def engine(cfg, seed=5, scale=1.0, **kw):
    from ghassan_b200.inference.engine import InferenceEngine
    from ghassan_b200.models.config import init_parameters
    named = init_parameters(cfg, seed)
    for k in named:
        if not k.endswith("norm"):
            named[k] = named[k] * scale
    return InferenceEngine(cfg, named, kv_cache="q8", **{**dict(fmt="f16", batch=1, max_len=400, prefill_chunk=128), **kw}), named


def ids_of(B, n, seed):
    return torch.randint(16, 512, (B, n), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("over,kw", [({}, {}), (dict(use_moe=False, use_qk_norm=False), {}), (dict(rope_type=1), dict(gemm_min_batch=2)), ({}, dict(fused_step=False)),
                                     (dict(sliding_window=9), {})])
def test_logits_follow_the_fp32_model(over, kw, monkeypatch):
    """The fp32 model with keys and values held as the pages hold them, token by token.  What is left is the engine's own 16-bit rounding (2^-11 of a key moves one
    code in fifty, the rest are the same), for which the bound is the one of the 16-bit cache's test.  A router's choice is not continuous: with hidden
    numbers off by 0.3 % router logits of about 2 are off by 0.006, the difference of two probabilities (each at most a quarter as steep) by 0.003; a sequence
    is compared up to the first token where the second and the third expert are nearer than twice that, in the plain model."""
    from ghassan_b200.models import reference
    cfg = cfg_of(**over)
    eng, named = engine(cfg, 11, 4.0, batch=2, **kw)

    def held(q, k, v, B, T, scale, window=0, segment_ids=None):
        seq, out = Seq(k.shape[1], k.shape[2]), []
        for t in range(T):
            seq.append(k[t:t + 1].numpy(), v[t:t + 1].numpy())
            kk, vv = seq.held()
            out.append(attention(q[t:t + 1].double().numpy(), kk, vv, t, scale, window)[0])
        return torch.from_numpy(np.concatenate(out)).float().reshape(plain(q, k, v, B, T, scale, window, segment_ids).shape)

    def watched(*args):
        probs, idx, w = route(*args)
        top = probs.sort(1, descending=True).values
        margins.append(top[:, 1] - top[:, 2])
        return probs, idx, w

    plain, route, margins = reference.attention, reference.route, []
    ref = reference.TorchModel(cfg, "cpu")
    ref.load_named(named)
    seq = ids_of(2, 24, 3)
    eng.reset(1)
    want, clear = [], []
    with torch.no_grad():
        for b in range(2):
            monkeypatch.setattr(reference, "route", watched)
            margins.clear()
            ref.logits(seq[b], 1, 24)
            near = (torch.stack(margins).amin(0) < 0.006).nonzero() if margins else []
            clear.append(int(near[0]) if len(near) else 24)
            monkeypatch.setattr(reference, "attention", held)
            want.append(ref.logits(seq[b], 1, 24))
            monkeypatch.setattr(reference, "attention", plain)
    assert sum(clear) >= 8, clear
    for j in range(24):
        eng.cur_tok.copy_(seq[:, j])
        eng._forward_token()
        got = eng.logits.cpu()
        for b in range(2):
            err = float((got[b] - want[b][j]).abs().max())
            assert j >= clear[b] or err < 0.03 * float(want[b][j].abs().max()) + 0.03, (j, b, err)
    eng.check()


@pytest.mark.parametrize("B,kw", [(1, {}), (2, {}), (2, dict(gemm_min_batch=2)), (1, dict(compute_dtype=torch.bfloat16))])
def test_a_prompt_in_portions_equals_token_by_token(B, kw):
    """300 tokens through portions of 128, 128 and the rest step by step, against 300 steps.  Pages that grow token by token are rounded again (one step instead of
    a half), and bfloat16 rows round 2^-8 where float16 rounds 2^-11."""
    cfg = cfg_of()
    prompt = ids_of(B, 300, 4)
    a, _ = engine(cfg, batch=B, **kw)
    a.reset(1)
    a.prefill(prompt)
    assert a.pos.tolist() == [300] * B and a._len == 300
    b, _ = engine(cfg, batch=B, **kw)
    b.reset(1)
    for j in range(300):
        b.cur_tok.copy_(prompt[:, j])
        b._forward_token()
    a.check()
    tol = 5e-2 if kw.get("compute_dtype") is None else 2e-1
    assert torch.allclose(a.logits, b.logits, rtol=tol, atol=tol), float((a.logits - b.logits).abs().max())
    assert a.state[:, :3].cpu().tolist() == b.state[:, :3].cpu().tolist()


def test_prompts_replay_and_generations_are_the_same_again():
    """Captured prompt passes and token steps against an engine's first, eager ones; pages of an earlier text do not show."""
    from ghassan_b200.inference.engine import SamplingParams
    cfg = cfg_of()
    sp = SamplingParams(greedy=True, repetition_penalty=1.0)
    a, _ = engine(cfg, batch=2)
    for n in (100, 260, 70, 333):
        prompt = ids_of(2, n, n)
        out = []
        for eng, graph in ((a, True), (engine(cfg, batch=2)[0], False)):
            eng.reset(1)
            eng.set_stop_tokens([])
            eng.prefill(prompt)
            first = eng.logits.clone()
            eng.sample_first(sp)
            eng.decode_steps(20, sp, use_graph=graph)
            eng.check()
            out.append((first, eng.transcript(21)))
        assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1]), n


def test_limits_are_refused():
    from ghassan_b200.inference.engine import InferenceEngine, SamplingParams
    from ghassan_b200.inference.generator import Generator
    cfg = cfg_of()
    eng, named = engine(cfg, max_len=100)
    sp = SamplingParams(greedy=True, repetition_penalty=1.0)
    assert eng.token_limit == 100
    with pytest.raises(ValueError, match="sized for 100"):
        eng.prefill(ids_of(1, 101, 1))
    eng.reset(1)
    eng.prefill(ids_of(1, 90, 1))
    eng.sample_first(sp)
    eng.decode_steps(10, sp)
    with pytest.raises(ValueError, match="exceed the 100"):
        eng.decode_steps(1, sp)
    with pytest.raises(ValueError, match="exceed the 100"):
        eng._forward_token()
    eng.check()
    res = Generator(eng).generate([ids_of(1, 95, 2)[0].tolist()], max_new_tokens=64, sampling=sp, stop_tokens=[])
    assert len(res.tokens[0]) == 6                            # five more tokens fit, and the last logits give one more
    with pytest.raises(ValueError, match="16bit or q8"):
        InferenceEngine(cfg, named, kv_cache="q4")


def test_the_command_line_takes_the_cache(tmp_path, capsys):
    from ghassan_b200.cli import infer as I
    from ghassan_b200.formats.gguf import export_gguf
    from ghassan_b200.models.config import init_parameters
    gold = os.path.join(os.path.dirname(__file__), "golden", "formats")
    cfg = cfg_of(vocab_size=400, hidden_size=128)
    path = str(tmp_path / "m.gguf")
    export_gguf(path, cfg, init_parameters(cfg, 22), os.path.join(gold, "tiny400.gtok"), "q8_k")
    args = ["--model", path, "--kv-cache", "q8"]
    assert I.main(["generate", *args, "--prompt", "salam", "--max-tokens", "8", "--seed", "3", "--no-stream", "--stats", "--ctx", "64"]) == 0
    assert "decode" in capsys.readouterr().out
    assert I.main(["bench", *args, "--prompt-tokens", "200", "--tokens", "24", "--greedy"]) == 0
    assert json.loads(capsys.readouterr().out.strip().splitlines()[-1])["decode_tokens_per_s"] > 0
    assert I.main(["perplexity", *args, "--text", "salam labas 3lik", "--ctx", "64"]) == 0
    with pytest.raises(SystemExit, match="16bit or q8"):
        I.main(["bench", "--model", path, "--kv-cache", "q3"])
