"""beam_search against a plain beam search that copies whole states and takes 64-bit log-softmax values of the same logits:
the same tokens, scores within 1e-5 (each of the n summed log-probabilities is within 2e-6 of its 64-bit value)."""
import numpy as np
import pytest
import torch

from yggdrasil_b200 import synth

pytestmark = pytest.mark.gpu


def plain(model, x, n, width, head=None, end=None):
    rows = len(x)
    state = model.init_state(rows)
    for t in range(x.shape[1]):
        logits, state = model.step(x[:, t], state)
    if head is not None:
        logits = head(state)
    beams = [[(0.0, list(x[r]), state[r], logits[r], False)] for r in range(rows)]
    for i in range(n):
        for r in range(rows):
            found = []
            for b, (score, toks, st, lg, done) in enumerate(beams[r]):
                logp = torch.log_softmax(lg.double(), -1).cpu().numpy()
                if done:
                    found.append((-score, b, 0, end, score, done))
                else:
                    found += [(-(score + logp[k]), b, k, k, score + logp[k], False) for k in range(len(logp))]
            found.sort(key=lambda f: f[:3])
            beams[r] = [(s, beams[r][b][1] + [k], beams[r][b][2], None, d or k == end)
                        for _, b, _, k, s, d in found[:width]]
        states = torch.stack([b[2] for r in beams for b in r])
        logits, new = model.step(np.array([b[1][-1] for r in beams for b in r], np.int32), states)
        if head is not None:
            logits = head(new)
        new, logits = new.view(rows, width, *new.shape[1:]), logits.view(rows, width, -1)
        beams = [[(s, k, new[r, j], logits[r, j], d) for j, (s, k, _, _, d) in enumerate(beams[r])] for r in range(rows)]
    return (np.array([[b[1] for b in r] for r in beams]), np.array([[b[0] for b in r] for r in beams]))


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    from yggdrasil_b200 import Yggdrasil
    from yggdrasil_b200.float_backend import B200FloatYggdrasil
    path = tmp_path_factory.mktemp("beam") / "m.bin"
    synth.write_random_model(synth.ModelShape(64, 8, 5, 27, 3, 8, 16), path, seed=3)
    layers, bias = synth.random_float_layers(dict(vocab=40, n=64, block=8, depth=5, readout=8, layer_input=16,
                                                  input_rank=16, router_token=8, routed=2), seed=5)
    return {"int8": Yggdrasil.load(path, backend="b200"), "float": B200FloatYggdrasil(layers, bias)}


@pytest.mark.parametrize("which", ["int8", "float"])
@pytest.mark.parametrize("rows,width,n", [(1, 1, 5), (1, 4, 12), (3, 5, 9), (2, 27, 4)])
def test_same_beams_as_a_plain_search(models, which, rows, width, n):
    from yggdrasil_b200.beam import beam_search
    model = models[which]
    x = np.random.default_rng(rows).integers(0, model.vocab, (rows, 6))
    tokens, scores = beam_search(model, x, n, width)
    want, best = plain(model, x, n, width)
    assert tokens.shape == (rows, width, 6 + n) and np.array_equal(tokens, want)
    np.testing.assert_allclose(scores, best, rtol=0, atol=1e-5)


@pytest.mark.parametrize("which", ["int8", "float"])
def test_with_a_head_on_the_states(models, which):
    from yggdrasil_b200 import quantize_rows
    from yggdrasil_b200.beam import beam_search, state_head
    model = models[which]
    k = model.layers * model.n
    g = torch.Generator().manual_seed(1)
    w = quantize_rows((torch.randn(model.vocab, k, generator=g) * (0.002 if which == "int8" else 0.2)).cuda())
    head = state_head(w.codes, w.scale, torch.randn(model.vocab, generator=g).cuda())
    x = np.random.default_rng(8).integers(0, model.vocab, (2, 3))
    tokens, scores = beam_search(model, x, 7, 4, head=head)
    want, best = plain(model, x, 7, 4, head=head)
    assert np.array_equal(tokens, want)
    np.testing.assert_allclose(scores, best, rtol=0, atol=1e-5)


def test_beams_that_end_keep_their_score(models):
    from yggdrasil_b200.beam import beam_search
    model = models["int8"]
    x = np.random.default_rng(9).integers(0, model.vocab, (3, 4))
    end = int(beam_search(model, x, 1, 3)[0][0, 1, -1])   # a token that some beams reach
    tokens, scores = beam_search(model, x, 10, 3, end=end)
    want, best = plain(model, x, 10, 3, end=end)
    assert np.array_equal(tokens, want) and (tokens[:, :, -1] == end).any()
    np.testing.assert_allclose(scores, best, rtol=0, atol=1e-5)


def test_one_row_no_tokens_and_refusals(models):
    from yggdrasil_b200.beam import beam_search
    model = models["int8"]
    tokens, scores = beam_search(model, [1, 2, 3], 5, 2)
    both, _ = beam_search(model, [[1, 2, 3]], 5, 2)
    assert tokens.shape == (2, 8) and np.array_equal(tokens, both[0])
    # width 1 is greedy decoding
    np.testing.assert_array_equal(beam_search(model, [4, 5], 6, 1)[0][0], model.generate([4, 5], 6, temperature=0))
    tokens, scores = beam_search(model, [1, 2], 0, 3)
    assert tokens.shape == (3, 2) and not scores.any()
    for args, kw in ((([1], 3, 28), {}), (([1], -1, 2), {}), (([1], 2, 0), {}), (([], 2, 2), {}), (([1], 2, 2), {"end": 27}),
                     (([99], 2, 2), {})):
        with pytest.raises(ValueError):
            beam_search(model, *args, **kw)


class GaveUp:
    """The library as after a product that gave up a wait."""
    def ygg_linear_status(self, index, stream, out):
        out._obj.value = -8   # YGG_E_TIMEOUT
        return 0


def test_a_head_whose_product_gave_up_is_reported(models, monkeypatch):
    from yggdrasil_b200 import _native, linear, quantize_rows
    from yggdrasil_b200.beam import beam_search, state_head
    model = models["int8"]
    w = quantize_rows(torch.randn(model.vocab, model.layers * model.n).cuda())
    head = state_head(w.codes, w.scale)
    monkeypatch.setattr(linear, "ops", GaveUp)
    for n in (0, 3):
        with pytest.raises(_native.YggError) as e:
            beam_search(model, [1, 2, 3], n, 2, head=head)
        assert e.value.code == _native.YGG_E_TIMEOUT
    beam_search(model, [1, 2, 3], 3, 2)   # no product of the operators in it
