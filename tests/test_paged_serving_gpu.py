"""What serves text over 8-bit pages beside ``generate``: scoring, throughput, the logits of a prompt."""
import os

import numpy as np
import pytest
import torch

from test_paged_engine_gpu import cfg_of, engine, ids_of

pytestmark = pytest.mark.gpu


def spoilt(cfg):
    """Parameters whose keys pass float16: a row of 256 normed numbers times weights of about 3000 is about 3000 * 16."""
    from ghassan_b200.models.config import init_parameters
    named = init_parameters(cfg, 5)
    hit = [k for k in named if k.endswith(("wk", "k_proj"))]
    assert hit, sorted(named)[:20]
    for k in hit:
        named[k] = np.random.default_rng(0).standard_normal(named[k].shape).astype(np.float32) * 3000
    return named


@pytest.mark.parametrize("what", ["perplexity", "benchmark", "generate"])
def test_keys_that_the_pages_cannot_hold_are_told(what):
    """Held as zero, so every number that comes out is finite and wrong; the next call on the device is not told of it."""
    from ghassan_b200.inference.engine import InferenceEngine
    from ghassan_b200.inference.generator import Generator
    cfg = cfg_of(use_qk_norm=False, use_moe=False)
    bad = Generator(InferenceEngine(cfg, spoilt(cfg), fmt="f16", batch=1, max_len=200, prefill_chunk=128, kv_cache="q8"))
    good = Generator(engine(cfg)[0])
    ids = ids_of(1, 40, 2)[0].tolist()

    def run(gen):
        if what == "perplexity":
            return gen.perplexity(ids)
        if what == "benchmark":
            return gen.benchmark(100, 20)
        return gen.generate([ids], max_new_tokens=8, stop_tokens=[])

    with pytest.raises(RuntimeError, match="303"):
        run(bad)
    assert run(good) is not None


def test_the_logits_command_tells_too(tmp_path, capsys):
    from ghassan_b200.cli import infer as I
    from ghassan_b200.formats.gguf import export_gguf
    from ghassan_b200.models.config import init_parameters
    gold = os.path.join(os.path.dirname(__file__), "golden", "formats")
    cfg = cfg_of(vocab_size=400, hidden_size=128, use_qk_norm=False, use_moe=False)
    for name, named, why in (("bad", spoilt(cfg), "303"), ("good", init_parameters(cfg, 5), None)):
        path = str(tmp_path / (name + ".gguf"))
        export_gguf(path, cfg, named, os.path.join(gold, "tiny400.gtok"), "q8_k")
        args = ["logits", "--model", path, "--kv-cache", "q8", "--ctx", "64", "--ids", "20 21 22 23 24"]
        if why:
            with pytest.raises(RuntimeError, match=why):
                I.main(args)
            assert "  " not in capsys.readouterr().out        # no table of wrong numbers
        else:
            assert I.main(args) == 0 and len(capsys.readouterr().out.splitlines()) >= 10
