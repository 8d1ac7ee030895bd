"""PagedEngine against the Hugging Face forward in float64 on the CPU, and the
example that serves candidates with it."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

# max-abs normalised error of fp32 logits: the decode engine's bar
TOL = 1e-5


def _model(model_type, hd=64, layers=2):
    torch.manual_seed(3)
    kw = dict(vocab_size=300, hidden_size=256, intermediate_size=384, num_hidden_layers=layers,
              num_attention_heads=4, num_key_value_heads=2, head_dim=hd, max_position_embeddings=256)
    if model_type == "llama":
        from transformers import LlamaConfig, LlamaForCausalLM

        m = LlamaForCausalLM(LlamaConfig(**kw))
    else:
        from transformers import Qwen3Config, Qwen3ForCausalLM

        m = Qwen3ForCausalLM(Qwen3Config(**kw))
        for layer in m.model.layers:
            for w in (layer.self_attn.q_norm.weight, layer.self_attn.k_norm.weight):
                torch.nn.init.normal_(w, 1.0, 0.2)
    return m.float().eval()


def _err(got, want):
    got = got.double().cpu()
    return float((got - want).abs().max() / want.abs().max())


@pytest.mark.parametrize("model_type,hd", [("llama", 64), ("qwen3", 128)])
def test_logits_match_the_full_forward(model_type, hd, gpu_device):
    from ssalaad_amd import PagedEngine

    m = _model(model_type, hd)
    ref = _model(model_type, hd).double()

    def want(ids):
        with torch.no_grad():
            return ref(torch.tensor([ids])).logits[0]

    eng = PagedEngine(m.to(gpu_device), max_seqs=5, pages=40, page=16)
    g = torch.Generator().manual_seed(0)
    text = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (37, 1, 90)]
    got = eng.feed([0, 2, 4], text, all_logits=True)
    assert _err(got, torch.cat([want(t) for t in text])) <= TOL
    text = {0: text[0], 2: text[1], 4: text[2]}

    def steps(seqs, n):
        for _ in range(n):
            tok = torch.randint(0, 300, (len(seqs),), generator=g)
            got = eng.step(seqs, tok)
            for s, t in zip(seqs, tok.tolist()):
                text[s] = text[s] + [t]
            assert _err(got, torch.stack([want(text[s])[-1] for s in seqs])) <= TOL

    steps([4, 0, 2], 3)
    eng.fork([0, 4], [1, 3])  # 40 positions: a shared page, half a copied one; 93: odd
    text[1], text[3] = text[0], text[4]
    steps([0, 1, 2, 3, 4], 20)
    eng.free([0, 4])
    used = int((eng.refs > 0).sum())
    assert int(eng.compact()) == used and int((eng.refs[:used] > 0).sum()) == used
    steps([1, 2, 3], 5)
    # a further chunk of a sequence beside another's first one
    more, new = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (21, 50)]
    got = eng.feed([3, 0], [more, new])
    text[3], text[0] = text[3] + more, new
    assert _err(got, torch.stack([want(text[3])[-1], want(new)[-1]])) <= TOL
    # prompt scores
    tokens = torch.randint(0, 300, (30,), generator=g)
    got = eng.score(4, tokens, top=4)
    lp = torch.log_softmax(want(tokens.tolist()), -1)[:-1]
    assert torch.allclose(got.logprobs.double().cpu(), lp.gather(1, tokens[1:, None])[:, 0], atol=1e-4)
    top = lp.topk(4)
    assert torch.allclose(got.top_logprobs.double().cpu(), top.values, atol=1e-4)
    assert torch.allclose(got.entropy.double().cpu(), -(lp.exp() * lp).sum(-1), atol=1e-4)
    # every page is given back
    eng.free([0, 1, 2, 3, 4])
    assert int(eng.refs.abs().sum()) == 0 and int((eng.table != -1).sum()) == 0


def test_a_window_bounds_what_the_engine_sees(gpu_device):
    """Against the forward with the same mask: the last 20 positions, the first 3."""
    from ssalaad_amd import PagedEngine

    m, ref = _model("llama"), _model("llama").double()
    eng = PagedEngine(m.to(gpu_device), max_seqs=1, pages=8, page=16, window=20, sinks=3)
    ids = torch.randint(0, 300, (70,), generator=torch.Generator().manual_seed(1))
    i, j = torch.arange(70)[:, None], torch.arange(70)[None]
    see = (j <= i) & ((j > i - 20) | (j < 3))
    mask = torch.where(see, 0.0, float("-inf")).double()[None, None]
    with torch.no_grad():
        want = ref(ids[None], attention_mask=mask).logits[0]
    assert _err(eng.feed([0], [ids[:60]], all_logits=True), want[:60]) <= TOL
    for t in range(60, 70):
        assert _err(eng.step([0], ids[t: t + 1]), want[t: t + 1]) <= TOL


def test_engine_refusals(gpu_device):
    from ssalaad_amd import PagedEngine

    eng = PagedEngine(_model("llama").to(gpu_device), max_seqs=3, pages=4, page=16)
    with pytest.raises(ValueError):
        eng.feed([0, 0], [[1], [2]])
    with pytest.raises(ValueError):
        eng.feed([3], [[1]])
    with pytest.raises(ValueError):
        eng.feed([0], [[]])
    with pytest.raises(ValueError):
        eng.feed([0], [list(range(257))])
    with pytest.raises(RuntimeError, match="free"):
        eng.feed([0], [[1] * 70])
    eng.feed([0], [[1] * 40])
    with pytest.raises(ValueError):
        eng.fork([1], [0])
    with pytest.raises(ValueError):
        eng.score(0, [1, 2])
    eng.fork([0], [1])  # takes the last free page
    with pytest.raises(RuntimeError):
        eng.fork([0], [2])
    with pytest.raises(ValueError):
        eng.step([0, 1], torch.tensor([1]))


def test_the_example_serves_candidates(gpu_device):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import serve_paged
    from ssalaad_amd import PagedEngine

    eng = PagedEngine(_model("llama").to(gpu_device), max_seqs=7, pages=60, page=16)
    prompt = list(range(40))
    tokens, logprobs = serve_paged.candidates(eng, prompt, n=6, new_tokens=20, every=4)
    assert tokens.shape == (6, 20) and bool((logprobs.diff() <= 0).all())
    again = torch.stack([
        eng.score(6, torch.cat([torch.tensor(prompt), t.cpu()])).logprobs[-20:].sum()
        for t in tokens[:1]])
    # 20 fp32 log probabilities of logits within the tolerance of each other
    assert torch.allclose(again, logprobs[:1], atol=20 * 1e-4)


def test_tokens_without_an_embedding(gpu_device):
    """Refused where the host can see them, a zero row where only the device can; never
    an index past the embeddings."""
    from ssalaad_amd import PagedEngine

    eng = PagedEngine(_model("llama").to(gpu_device), max_seqs=2, pages=8, page=16)
    for bad in ([5, 300], [-1], torch.tensor([2 ** 40])):
        with pytest.raises(ValueError, match="token ids"):
            eng.feed([0], [bad])
        with pytest.raises(ValueError, match="token ids"):
            eng.score(0, bad)
    with pytest.raises(ValueError, match="token ids"):
        eng.step([0], torch.tensor([300]))
    assert int(eng.lengths.abs().sum()) == 0 and int(eng.refs.abs().sum()) == 0
    ids = torch.tensor([7, 300, -5, 2 ** 40], device=gpu_device)
    got = eng.feed([0], [ids], all_logits=True)
    assert bool(got.isfinite().all())
    alone = eng.feed([1], [[7]])
    assert _err(got[:1], alone.double().cpu()) <= TOL
    # the first row is the embedding's, the others are zeros
    h, x = eng._embed_rmsnorm(ids, eng.layers[0].in_norm)
    assert torch.equal(h[0], eng.embed[7]) and not h[1:].any() and not x[1:].any()


def test_int32_tokens_step(gpu_device):
    from ssalaad_amd import PagedEngine

    eng = PagedEngine(_model("llama").to(gpu_device), max_seqs=2, pages=8, page=16)
    a = eng.step([0], torch.tensor([9], dtype=torch.int32))
    b = eng.step([1], torch.tensor([9], device=gpu_device))
    assert torch.equal(a, b)


@pytest.mark.parametrize("where", ["the lm head", "a layer"])
def test_a_call_that_fails_changes_no_sequence(where, gpu_device):
    """Nothing grows, no page is lost, and the call can be made again."""
    from ssalaad_amd import PagedEngine

    m = _model("llama").to(gpu_device)
    eng = PagedEngine(m, max_seqs=4, pages=12, page=16)
    ref = PagedEngine(m, max_seqs=4, pages=12, page=16)

    def fail(*a):
        raise torch.OutOfMemoryError("no memory")

    def failing(call):
        head, down = eng.lm_head, eng.layers[1].down
        if where == "a layer":
            eng.layers[1].down = fail
        else:
            eng.lm_head = fail
        with pytest.raises(torch.OutOfMemoryError):
            call()
        eng.lm_head, eng.layers[1].down = head, down

    text = list(range(40))
    failing(lambda: eng.feed([0, 2], [text, text[:17]]))
    assert int(eng.lengths.sum()) == 0
    assert torch.equal(eng.feed([0, 2], [text, text[:17]]), ref.feed([0, 2], [text, text[:17]]))
    assert int(eng.refs.sum()) == 5
    for t in range(12):  # across a page's end
        tok = torch.tensor([t, t + 1])
        failing(lambda: eng.step([0, 2], tok))
        assert torch.equal(eng.step([0, 2], tok), ref.step([0, 2], tok))
    assert torch.equal(eng.lengths, ref.lengths) and int(eng.refs.sum()) == int(ref.refs.sum())
    # a fork into a sequence that a failed call reserved pages for
    failing(lambda: eng.feed([1], [text]))
    eng.fork([0], [1])
    ref.fork([0], [1])
    tok = torch.tensor([3])
    assert torch.equal(eng.step([1], tok), ref.step([1], tok))
    assert int(eng.refs.sum()) == int(ref.refs.sum())
    failing(lambda: eng.feed([3], [text[:20]]))
    eng.free([0, 1, 2, 3])
    assert int(eng.refs.abs().sum()) == 0 and int((eng.table != -1).sum()) == 0


def test_forks_of_no_such_sequence_are_refused(gpu_device):
    from ssalaad_amd import PagedEngine

    eng = PagedEngine(_model("llama").to(gpu_device), max_seqs=3, pages=8, page=16)
    eng.feed([2], [[1, 2, 3]])
    for src, dst in (([-1], [0]), ([3], [0]), ([2], [0, 1]), ([2, 2], [0])):
        with pytest.raises(ValueError):
            eng.fork(src, dst)
    assert eng.lengths.tolist() == [0, 0, 3] and int(eng.refs.sum()) == 1
    eng.fork([2, 2], [0, 1])
    assert eng.lengths.tolist() == [3, 3, 3] and int(eng.refs.sum()) == 3


def test_the_engine_runs_on_its_models_device(gpu_device, monkeypatch):
    """Every call makes the model's device current for its launches."""
    from ssalaad_amd import PagedEngine

    entered = []

    class Device(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    eng = PagedEngine(_model("llama").to(gpu_device), max_seqs=3, pages=8, page=16)
    monkeypatch.setattr(torch.cuda, "device", Device)
    for call in (lambda: eng.feed([0], [[1, 2]]), lambda: eng.step([0], torch.tensor([3])),
                 lambda: eng.fork([0], [1]), lambda: eng.free([0]), lambda: eng.compact(),
                 lambda: eng.score(2, [1, 2, 3])):
        entered.clear()
        call()
        assert entered and set(entered) == {gpu_device.index}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("model_type,hd", [("llama", 64), ("qwen3", 128)])
def test_logits_in_16_bits(model_type, hd, dtype, gpu_device):
    """A prompt, steps, a fork and a further chunk. Two layers round some ten times on
    the way to the logits: within 16 roundings of the forward in float64 of the same
    (rounded) weights, relative to the largest logit."""
    from ssalaad_amd import PagedEngine

    m = _model(model_type, hd).to(dtype)
    ref = _model(model_type, hd).to(dtype).double()
    eng = PagedEngine(m.to(gpu_device), max_seqs=3, pages=30, page=16)
    g = torch.Generator().manual_seed(4)
    text = torch.randint(0, 300, (90,), generator=g)
    with torch.no_grad():
        want = ref(text[None]).logits[0]
    tol = 16 * torch.finfo(dtype).eps / 2
    assert _err(eng.feed([0], [text[:61]], all_logits=True), want[:61]) <= tol
    for t in range(61, 66):
        assert _err(eng.step([0], text[t: t + 1]), want[t: t + 1]) <= tol
    eng.fork([0], [2])
    got = eng.feed([2, 0], [text[66:], text[66:70]], all_logits=True)
    assert _err(got, torch.cat([want[66:], want[66:70]])) <= tol


@pytest.mark.parametrize("model_type,kv", [("llama", 4), ("llama", 2), ("qwen3", 2)])
@pytest.mark.parametrize("dtype,nm", [(torch.float32, False), (torch.bfloat16, False),
                                      (torch.bfloat16, True)])
def test_a_compressed_model_is_served(model_type, kv, dtype, nm, gpu_device):
    """SLR projections: a prompt, steps of two sequences, a fork and a further chunk,
    against the dense twin in float64. fp32: the decode engine's bar; bf16: twice the
    error of the reference module's own arithmetic, or 3e-2. (2:4 S is 16-bit.)"""
    from ssalaad_amd import PagedEngine
    from test_gpu_decode import _slr_triple

    model, dense, mirror = _slr_triple(model_type, dtype, kv, gpu_device, seed=5, nm=nm)
    eng = PagedEngine(model.to(gpu_device).eval(), max_seqs=3, pages=30, page=16)
    g = torch.Generator().manual_seed(6)
    text = torch.randint(0, 384, (100,), generator=g)
    with torch.no_grad():
        want = dense.eval()(text[None]).logits[0]
        tol = TOL if dtype == torch.float32 else min(
            3e-2, 2 * _err(mirror(text[None]).logits[0], want))
    got = [eng.feed([0], [text[:70]], all_logits=True)]
    for t in range(70, 80):
        got.append(eng.step([0], text[t: t + 1]))
    eng.fork([0], [2])
    got.append(eng.feed([2, 0], [text[80:], text[80:85]], all_logits=True))
    assert _err(torch.cat(got), torch.cat([want, want[80:85]])) <= tol
