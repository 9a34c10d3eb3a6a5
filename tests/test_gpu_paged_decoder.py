"""The operators of a batched step together: LlamaDecoder.step_paged and generate_batch against the float64 model with the same
storage rule (oracle/paged_ref.py). As for the other int8 cache, logits are held to 5e-3 of the largest: a code next to a
rounding border may differ by one from the float64 model's; greedy tokens are compared where the model's choice is
clearer than that."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TOL = 5e-3


def build(seed, block=16, seqs=3, heads=4, kv=2, dim=32):
    from grilly2_b200.infer import llama
    from oracle.paged_ref import PagedDecoderRef
    cfg = llama.LlamaConfig(vocab_size=500, hidden_size=128, num_hidden_layers=3, num_attention_heads=heads, num_key_value_heads=kv, head_dim=dim,
                            intermediate_size=256, max_cache_len=96)
    w = llama.random_weights(cfg, seed=seed, sigma=0.08)
    cos, sin = llama.rotary_tables(cfg)
    return cfg, llama.LlamaDecoder(cfg, w), lambda n=seqs: PagedDecoderRef(cfg, w, cos, sin, n, block)


def dev(a):
    from grilly2_b200 import _C
    return _C.Tensor.from_numpy(np.ascontiguousarray(a, dtype=np.int32))


@pytest.mark.parametrize("block,heads,kv,dim", [(16, 4, 2, 32), (32, 6, 1, 64), (64, 2, 2, 128)])
def test_mixed_steps_equal_the_float64_model(block, heads, kv, dim):
    """Prompts, single tokens, requests that join late or pause, padded rows, a request released and begun again."""
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    cfg, model, make = build(21, block, heads=heads, kv=kv, dim=dim)
    ref, rng = make(), np.random.default_rng(2)
    cache = PagedKvCache.for_model(cfg, seqs=3, blocks=3 * -(-96 // block), block_size=block)
    for i, counts in enumerate([[20, 0, 3], [1, 37, 1], [1, 1, 1], [0, 1, 18], [1, 1, 1]]):
        new = [list(rng.integers(0, 500, c)) for c in counts]
        pad = (0, 2, 5)[i % 3]
        step = PagedStep(cache, sum(counts) + pad)
        cache.plan(dev(counts), step)
        got = model.step_paged(dev([t for r in new for t in r] + [0] * pad), cache, step, max_count=max(counts)).numpy()
        for b, want in enumerate(ref.step(new)):
            if want is None:
                assert np.isnan(got[b]).all()
                continue
            worst = np.abs(got[b] - want).max() / np.abs(want).max()
            print(f"[paged decoder] step {i} request {b}: {worst:.2e} of the largest logit")
            assert worst <= TOL
        np.testing.assert_array_equal(cache.lengths(), ref.lens)
    cache.release(dev([0, 1, 0]))
    again = make(1)
    new = list(rng.integers(0, 500, 9))
    step = PagedStep(cache, 9)
    cache.plan(dev([0, 9, 0]), step)
    got, want = model.step_paged(dev(new), cache, step).numpy()[1], again.step([new])[0]
    assert np.abs(got - want).max() <= TOL * np.abs(want).max()


PROMPTS = [[5, 17, 99, 3, 42, 7, 64], [8], list(range(100, 140))]


@pytest.mark.parametrize("graphed", [True, False], ids=["graphed", "eager"])
def test_greedy_batch_follows_the_float64_model(graphed):
    from grilly2_b200.infer.generation import generate_batch
    cfg, model, make = build(22)
    got = generate_batch(model, PROMPTS, max_new_tokens=20, block_size=16, graphed=graphed)
    ref = make()
    new, clear = [list(p) for p in PROMPTS], 0
    for i in range(20):
        logits = ref.step(new)
        new = []
        for b, lg in enumerate(logits):
            tok = int(got[b][len(PROMPTS[b]) + i])
            assert lg[tok] >= lg.max() - 2 * TOL * np.abs(lg).max(), (i, b)  # the model's choice, or one as good
            clear += tok == int(np.argmax(lg))
            new.append([tok])
    assert clear >= 50  # of 60
    assert all(g.dtype == np.int64 and list(g[:len(p)]) == p and len(g) == len(p) + 20 for g, p in zip(got, PROMPTS))


def test_batch_equals_requests_on_their_own_and_ends_them():
    """Greedy requests do not depend on their neighbours; eos and max_length end each on its own."""
    from grilly2_b200.infer.generation import generate_batch
    cfg, model, _ = build(23)
    whole = generate_batch(model, PROMPTS, max_new_tokens=12)
    for p, w in zip(PROMPTS, whole):
        assert generate_batch(model, [p], max_new_tokens=12)[0].tolist() == w.tolist()
    eos = int(whole[0][len(PROMPTS[0]) + 3])
    cut = generate_batch(model, PROMPTS, max_new_tokens=12, eos_token_id=eos)
    for p, w, c in zip(PROMPTS, whole, cut):
        at = [i for i in range(len(p), len(w)) if w[i] == eos]
        assert c.tolist() == w[:at[0] + 1 if at else len(w)].tolist()
    assert [len(x) for x in generate_batch(model, PROMPTS, max_length=42)] == [42, 42, 42]
    assert [len(x) for x in generate_batch(model, PROMPTS, max_length=8)] == [8, 8, 40]


def test_sampled_batch_is_seeded_and_settings_are_per_request():
    from grilly2_b200.infer.generation import generate_batch
    from grilly2_b200.infer.sampling import Generator
    cfg, model, _ = build(24)
    kw = dict(max_new_tokens=10, do_sample=[True, False, True], temperature=[0.9, 1.0, 1.2], top_k=[5, 50, 0], top_p=[0.95, 1.0, 0.9], min_p=[0.0, 0.0, 0.05])
    a, b, c = (generate_batch(model, PROMPTS, generator=Generator(s), graphed=gr, **kw) for s, gr in ((7, True), (7, False), (8, True)))
    assert all(x.tolist() == y.tolist() for x, y in zip(a, b))
    assert a[0].tolist() != c[0].tolist() and a[2].tolist() != c[2].tolist()
    greedy = generate_batch(model, PROMPTS, max_new_tokens=10)
    assert a[1].tolist() == greedy[1].tolist()


def test_a_prompt_at_its_end_takes_no_room():
    """A request that asks for no token is returned as it is, whatever its length, beside others that go on."""
    from grilly2_b200.infer.generation import generate_batch
    cfg, model, _ = build(26)
    long, short = list(range(33)), [7, 8, 9]
    got = generate_batch(model, [long, short, [1] * 120], max_length=33, block_size=16)
    assert [len(x) for x in got] == [33, 33, 120] and got[0].tolist() == long
    assert got[1].tolist() == generate_batch(model, [short], max_length=33, block_size=16)[0].tolist()
    assert [x.tolist() for x in generate_batch(model, [long, short], max_new_tokens=0)] == [long, short]


def test_logits_that_are_no_numbers_end_the_batch():
    from grilly2_b200.infer.generation import generate_batch
    cfg, model, _ = build(27)
    with pytest.raises(RuntimeError, match="request 1"):
        generate_batch(model, [[3, 4], [500]], max_new_tokens=3)  # no such token


def test_refusals_of_the_batch():
    from grilly2_b200.infer.generation import generate_batch
    from grilly2_b200.infer.paged import PagedKvCache, PagedStep
    cfg, model, _ = build(25)
    with pytest.raises(ValueError, match="non-empty"):
        generate_batch(model, [[1], []], max_new_tokens=2)
    with pytest.raises(ValueError, match="one per prompt"):
        generate_batch(model, PROMPTS, max_new_tokens=2, top_k=[1, 2])
    with pytest.raises(ValueError, match="not used by the model"):
        generate_batch(model, PROMPTS, max_new_tokens=2, banana=1)
    with pytest.raises(NotImplementedError, match="use_cache"):
        generate_batch(model, PROMPTS, max_new_tokens=2, use_cache=False)
    with pytest.raises(NotImplementedError, match="repetition"):
        generate_batch(model, PROMPTS, max_new_tokens=2, repetition_penalty=1.2)
    with pytest.raises(ValueError, match="temperature"):
        generate_batch(model, PROMPTS, max_new_tokens=2, do_sample=True, temperature=0.0)
    with pytest.raises(RuntimeError, match="96 cached positions"):
        generate_batch(model, PROMPTS, max_new_tokens=80)
    with pytest.raises(RuntimeError, match="cannot hold the prompts"):
        generate_batch(model, PROMPTS, max_new_tokens=2, block_size=16, blocks=3)
    with pytest.raises(RuntimeError, match="has run out"):
        generate_batch(model, [[1] * 16, [2] * 16], max_new_tokens=20, block_size=16, blocks=3)
    cache = PagedKvCache(layers=1, kv_heads=2, head_dim=32, blocks=4, seqs=1, max_blocks=2, block_size=16)
    step = PagedStep(cache, 2)
    with pytest.raises(RuntimeError, match="the model has"):
        model.step_paged(dev([1, 2]), cache, step)
    with pytest.raises(RuntimeError, match="takes 2 int32 tokens"):
        model.step_paged(dev([1, 2, 3]), cache, step)
