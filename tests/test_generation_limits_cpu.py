"""Generation up to the last token that an engine's caches hold, over an engine of a few lines that counts its tokens as the paged one does."""
import pytest
import torch

from ghassan_b200.inference.engine import InferenceEngine
from ghassan_b200.inference.generator import Generator
from ghassan_b200.inference.token_loop import SamplingParams, TokenLoop

V = 40


class Counting:
    """What the generator needs of an engine; token t is followed by t + 1.  Tokens are counted by the real engine's rule."""
    host_only, paged = True, True

    def __init__(self, cap, batch=1):
        self.cap, self.B, self.passes, self.told = cap, batch, 0, []
        self.logits, self.cur_tok = torch.zeros(batch, V), torch.zeros(batch, dtype=torch.int32)
        self.tok_log = torch.zeros(batch, 1000)
        self._len = 0

    token_limit = InferenceEngine.token_limit
    _claim = InferenceEngine._claim

    def reset(self, seed=0):
        self._len = 0

    def set_stop_tokens(self, ids):
        pass

    def check(self, what="generation"):
        self.told.append(what)

    def prefill(self, ids):
        for j in range(ids.shape[1]):
            self.cur_tok.copy_(ids[:, j])
            self._forward_token()

    def _forward_token(self):
        self._claim(1)
        self.passes += 1
        self.logits.fill_(-10.0)
        for b in range(self.B):
            self.logits[b, (int(self.cur_tok[b]) + 1) % V] = 10.0


HOST = dict(temperature=0.01, top_p=1.0, min_p=0.0, repetition_penalty=1.0)


@pytest.mark.parametrize("sp", [SamplingParams(no_repeat_ngram=3, **HOST), SamplingParams(repetition_window=2000, **HOST), SamplingParams(top_k=0, **HOST)])
@pytest.mark.parametrize("cap,n,asked,got", [(10, 4, 64, 7), (10, 10, 5, 1), (10, 4, 7, 7), (10, 4, 6, 6), (10, 1, 64, 10)])
def test_the_host_sampler_generates_up_to_the_limit(sp, cap, n, asked, got):
    """cap - n tokens have a place after the prompt, and the last logits give one more, which needs none."""
    assert not sp.device_ok()
    eng = Counting(cap)
    res = Generator(eng).generate([list(range(n))], max_new_tokens=asked, sampling=sp, stop_tokens=[])
    assert res.tokens == [list(range(n, n + got))] and res.stopped == ["length"]
    assert eng.passes == n + got - 1 <= cap                   # no pass behind the last token


def test_a_sequence_that_stops_early_does_not_end_the_others():
    eng = Counting(12, batch=2)
    res = Generator(eng).generate([[0, 1], [5, 6]], max_new_tokens=64, sampling=SamplingParams(no_repeat_ngram=3, **HOST), stop_tokens=[4])
    assert res.tokens == [[2, 3], list(range(7, 18))] and res.stopped == ["eos", "length"] and eng.passes == 12


@pytest.mark.parametrize("graph", [True, False])
def test_no_steps_are_no_steps(graph):
    """With settings that no captured step has yet, too: the step that precedes a capture is one of those asked for."""
    class Loop(TokenLoop):
        graph, _graph_key, n_stop, ran = None, None, 0, 0

        def _draw_uniforms(self, n):
            pass

        def _step_eager(self, sp):
            self.ran += 1

    loop = Loop()
    loop.decode_steps(0, SamplingParams(greedy=True), use_graph=graph)
    assert loop.ran == 0 and loop.graph is None
    with pytest.raises(ValueError, match="host sampler"):
        loop.decode_steps(0, SamplingParams(top_k=0), use_graph=graph)


def test_scoring_asks_whether_the_cache_held_what_it_was_given():
    eng = Counting(50)
    nll, n = Generator(eng).score_tokens([1, 2, 3, 4])
    assert n == 3 and nll < 1e-3 and len(eng.told) == 1
    eng.paged = False                                         # the other engines have no such question
    Generator(eng).score_tokens([1, 2, 3, 4])
    assert len(eng.told) == 1
