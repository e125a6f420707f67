"""LMGenerator: tokens through the caches give the logits of the whole-sequence model; prefix, drafts and ragged batches.

Tolerances: float32 logits agree to 1e-3 of their largest magnitude (two orders of summation through two layers of
float32 kernels, each within 2e-4); fp16 to 3e-2, the tolerance that the model's own fp16 tests use; int8 adds the
codes' own step of 1/254 of each row's largest entry, and is held to 1e-1."""
import pytest
import torch

from first_passage_attention_b200.lm import FPALanguageModel, LMConfig, LMGenerator

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
CFG = LMConfig(vocab=211, d_model=64, n_heads=2, n_layers=2)


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")


def model(cfg=CFG, seed=0, scale=1.0):
    torch.manual_seed(seed)
    m = FPALanguageModel(cfg).cuda()
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(scale)
    return m


def whole(m, tokens, dtype):
    with torch.no_grad(), torch.autocast(device_type="cuda", dtype=F16, enabled=dtype == F16):
        return m(tokens).float()


@pytest.mark.parametrize("dtype,storage,tol", [(F32, None, 1e-3), (F16, None, 3e-2), (F16, torch.int8, 1e-1), (F32, torch.int8, 1e-1)])
def test_extend_gives_the_models_logits(dtype, storage, tol):
    m = model()
    tokens = torch.randint(0, CFG.vocab, (3, 90), generator=torch.Generator().manual_seed(1)).cuda()
    want = whole(m, tokens, dtype)
    gen = LMGenerator(m, 1000, page_size=32, dtype=dtype, storage=storage)
    gen.reset(3, 100)
    got, at = [gen.extend(tokens[:, :50], first=True)], 50
    gen.keep(torch.full((3,), 50, dtype=torch.int32, device="cuda"))
    for n in (1, 7, 16, 3, 13):
        got.append(gen.extend(tokens[:, at:at + n]))
        gen.keep(torch.full((3,), n, dtype=torch.int32, device="cuda"))
        at += n
    got = torch.cat(got, 1)
    assert (got - want).abs().max().item() <= tol * want.abs().max().item()
    # Drafts taken back: other tokens first, refused after two, then the right ones.
    gen.reset(3, 100)
    gen.extend(tokens[:, :50], first=True)
    gen.keep(torch.full((3,), 50, dtype=torch.int32, device="cuda"))
    wrong = tokens[:, 50:56].clone()
    wrong[:, 2:] = (wrong[:, 2:] + 1) % CFG.vocab
    gen.extend(wrong)
    gen.keep(torch.full((3,), 2, dtype=torch.int32, device="cuda"))
    again = gen.extend(tokens[:, 52:60])
    assert (again - want[:, 52:60]).abs().max().item() <= tol * want.abs().max().item()
    for c in gen.caches:
        c.check()


def test_extend_behind_a_prefix():
    m = model()
    g = torch.Generator().manual_seed(2)
    prefix = torch.randint(0, CFG.vocab, (70,), generator=g).tolist()
    own = torch.randint(0, CFG.vocab, (4, 20), generator=g).cuda()
    gen = LMGenerator(m, 1000, page_size=32, dtype=F32)
    gen.reset(4, 40, prefix)
    got = []
    for i in range(0, 20, 5):
        got.append(gen.extend(own[:, i:i + 5]))
        gen.keep(torch.full((4,), 5, dtype=torch.int32, device="cuda"))
    tokens = torch.cat([torch.tensor(prefix, device="cuda").expand(4, -1), own], 1)
    want = whole(m, tokens, F32)[:, 70:]
    assert (torch.cat(got, 1) - want).abs().max().item() <= 1e-3 * want.abs().max().item()


@pytest.mark.parametrize("with_prefix", [False, True])
@pytest.mark.parametrize("n_draft", [0, 1, 5])
def test_generate_follows_the_model(with_prefix, n_draft):
    """At a temperature near zero every token is the model's best after the tokens before it (to the logits' tolerance),
    whatever the draft proposes."""
    m = model(scale=1.5)
    small = LMConfig(vocab=CFG.vocab, d_model=32, n_heads=2, n_layers=1)
    draft = LMGenerator(model(small, seed=5), 2000, page_size=32, dtype=F32) if n_draft else None
    g = torch.Generator().manual_seed(3)
    prefix = torch.randint(0, CFG.vocab, (45,), generator=g).tolist() if with_prefix else None
    prompts = [torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in (1, 9, 40)]
    gen = LMGenerator(m, 2000, page_size=32, dtype=F32)
    out = gen.generate(prompts, 12, temperature=1e-4, prefix=prefix, draft=draft, n_draft=n_draft,
                       generator=torch.Generator(device="cuda").manual_seed(4))
    for prompt, new in zip(prompts, out):
        assert len(new) == 12
        seq = (prefix or []) + prompt + new
        logits = whole(m, torch.tensor([seq], device="cuda"), F32)[0]
        for i, t in enumerate(new):
            row = logits[len(seq) - 12 + i - 1]
            assert (row.max() - row[t]).item() <= 2e-3 * row.abs().max().item(), (len(prompt), i)


def test_a_model_that_drafts_for_itself_is_accepted():
    """With the model as its own draft, in float32, nearly every draft is accepted: n tokens take few rounds."""
    m = model()
    gen, draft = LMGenerator(m, 1000, page_size=32, dtype=F32), LMGenerator(m, 1000, page_size=32, dtype=F32)
    calls = []
    extend = gen.extend
    gen.extend = lambda *a, **k: (calls.append(1), extend(*a, **k))[1]
    out = gen.generate([[1, 2, 3], [4, 5]], 30, draft=draft, n_draft=5, generator=torch.Generator(device="cuda").manual_seed(6))
    assert all(len(x) == 30 for x in out)
    assert len(calls) <= 1 + 7  # the prompts, and 30 tokens at 6 a round with two to spare


def test_refusals():
    gen = LMGenerator(model(), 100, page_size=32, dtype=F32)
    with pytest.raises(ValueError, match="pages"):
        gen.reset(10, 100)
    gen.reset(1, 64)
    with pytest.raises(ValueError, match="at most 16"):
        gen.extend(torch.zeros(1, 17, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError, match="no prompt may be empty"):
        gen.generate([[]], 1)


def test_tokens_past_the_room_are_refused():
    """What `reset` has given no room for is refused, by the lengths as they are and not by what was fed and taken back."""
    gen = LMGenerator(model(), 200, page_size=32, dtype=F32)
    tokens = torch.zeros(2, 16, dtype=torch.long, device="cuda")
    for prefix in (None, list(range(40))):
        gen.reset(2, 60, prefix)  # two pages of 32 each
        for i in range(30):       # far more than 64 tokens, all taken back
            gen.extend(tokens)
            gen.keep(torch.zeros(2, dtype=torch.int32, device="cuda"))
        for _ in range(3):
            gen.extend(tokens)
            gen.keep(torch.tensor([5, 16], dtype=torch.int32, device="cuda"))
        gen.extend(tokens)
        gen.keep(torch.tensor([16, 15], dtype=torch.int32, device="cuda"))
        gen.extend(tokens[:, :1])
        with pytest.raises(ValueError, match="room"):
            gen.extend(tokens[:, :2])
    gen.reset(2, 60)
    with pytest.raises(ValueError, match="room"):
        gen.extend(torch.zeros(2, 65, dtype=torch.long, device="cuda"), first=True)
    gen.reset(2, 60)
    gen.extend(tokens)
    gen.keep(torch.ones(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="first"):
        gen.extend(tokens, first=True)
    gen.reset(2, 60, [1, 2, 3])
    with pytest.raises(ValueError, match="first"):
        gen.extend(tokens, first=True)
    with pytest.raises(ValueError, match="pages"):
        gen.reset(8, 0)  # each sequence holds a page
    for c in gen.caches:
        c.check()


def test_generate_raises_what_the_kernels_report():
    """A page id outside the pool, met while answering: no answer comes back."""
    for which in (0, 1):
        gen = LMGenerator(model(), 1000, page_size=32, dtype=F32)
        draft = LMGenerator(model(seed=2), 1000, page_size=32, dtype=F32)
        bad = (gen, draft)[which]
        start = bad._start

        def broken(*args):
            cur = start(*args)
            bad.table[0, 0] = 10 ** 6
            return cur

        bad._start = broken
        with pytest.raises(ValueError, match="outside"):
            gen.generate([[1, 2, 3], [4, 5]], 6, draft=draft, n_draft=2)


def test_keep_takes_no_more_than_was_fed():
    """Counts outside 0 .. n: an index past the walks would be a fault on the device."""
    gen = LMGenerator(model(), 400, page_size=32, dtype=F32)
    tokens = torch.arange(12, device="cuda").view(3, 4)
    walks = []
    for counts in ([4, 0, 2], [2 ** 31 - 1, -5, 2]):
        gen.reset(3, 60)
        gen.extend(tokens)
        gen.keep(torch.tensor(counts, dtype=torch.int32, device="cuda"))
        assert gen.lengths.tolist() == [4, 0, 2]
        walks.append(gen.walk)
    assert torch.equal(*walks)


def test_feeding_a_prompt_needs_no_logits():
    """Prompts and prefixes go into the caches without the output layer's [tokens, vocabulary] logits."""
    cfg = LMConfig(vocab=50304, d_model=64, n_heads=2, n_layers=1)
    gen = LMGenerator(model(cfg), 8000, page_size=64)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, cfg.vocab, (3000,), generator=g).tolist()
    torch.cuda.synchronize()
    for prompts, prefix in (([ids[:1500], ids[1500:]], None), ([ids[:40]], ids)):
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        gen.generate(prompts, 2, prefix=prefix)
        # The logits of one chunk of 16 tokens in fp16 and float32 are 5 MB, those of 3000 tokens 900 MB.
        assert torch.cuda.max_memory_allocated() - before < 100 * 2 ** 20


def test_generate_refusals():
    gen = LMGenerator(model(), 1000, page_size=32, dtype=F32)
    for temperature in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            gen.generate([[1]], 2, temperature=temperature)
    with pytest.raises(ValueError, match="draft"):
        gen.generate([[1]], 2, draft=gen)
    with pytest.raises(ValueError, match="prompt"):
        gen.generate([], 2)


def test_ids_outside_the_vocabulary_are_refused():
    """Raised on the host: on the device they would be faults."""
    gen = LMGenerator(model(), 1000, page_size=32, dtype=F32)
    for bad in (-1, CFG.vocab):
        with pytest.raises(ValueError, match="token ids"):
            gen.generate([[1, 2], [3, bad]], 2)
        with pytest.raises(ValueError, match="token ids"):
            gen.generate([[1, 2]], 2, prefix=[0, bad])
        with pytest.raises(ValueError, match="token ids"):
            gen.reset(1, 32, [bad])
    for vocab in (CFG.vocab - 1, CFG.vocab + 64):
        draft = LMGenerator(model(LMConfig(vocab=vocab, d_model=64, n_heads=2, n_layers=1)), 1000, page_size=32, dtype=F32)
        with pytest.raises(ValueError, match="vocabulary"):
            gen.generate([[1, 2]], 2, draft=draft)
    assert len(gen.generate([[1, CFG.vocab - 1]], 3, prefix=[0])[0]) == 3
