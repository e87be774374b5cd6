"""Llama and GPT-2 serving requests of different lengths over pages, against the same requests one by one over the model's own cache."""
import numpy as np
import pytest

from ruai_b200 import nn

pytestmark = pytest.mark.gpu

# Pages in f32 differ from the model's own cache in the order of sums only: the project's tolerance on logits.  In 16 bits every key, value,
# query and attention output is rounded to half a step (2^-11 or 2^-8) once in a layer; the logits of these two-layer models are sums of
# hundreds of such terms, whose errors add up like their squares: a few half steps of the logits' scale.
REL = {nn.F32: 1e-3, nn.F16: 8 * 2.0 ** -11, nn.BF16: 8 * 2.0 ** -8}


@pytest.fixture(scope="module")
def dev():
    assert nn.Device.is_available(), "these tests need a CUDA device"
    return nn.Device.cuda(0)


def llama(dev, H=8, KV=2, hd=64, V=500, d=256, ff=512, L=2, bits=8, positions=512):
    m = nn.Llama(dev, nn.LlamaConfig(V, d, ff, L, H, KV, hd, positions, 1e-5, 10000.0, 0))
    m.load_synthetic(5, bits, 32)
    return m


def gpt2(dev, V=500, positions=400, d=256, L=2, H=4):
    m = nn.GPT2(dev, nn.GPT2Config(V, positions, d, L, H))
    m.load_synthetic(6, 8, 32)
    return m


MODELS = {"llama": llama, "llama int4 hd 128": lambda dev: llama(dev, H=4, KV=1, hd=128, bits=4), "llama hd 80": lambda dev: llama(dev, H=6, KV=3, hd=80), "gpt2": gpt2}


def alone(m, ids):
    """Logits after the last of a request's tokens, by the model's own cache."""
    m.cache_clear()
    return m.forward_cached(np.asarray(ids)[None])[0]


@pytest.mark.parametrize("dtype", [nn.F32, nn.F16, nn.BF16])
@pytest.mark.parametrize("name", MODELS)
def test_steps_of_mixed_requests(dev, name, dtype):
    """Prompts, parts of a prompt and single tokens in one step; requests end, and others take their pages."""
    m = MODELS[name](dev)
    rng = np.random.default_rng(1)
    m.serve_start(40, 4, page=16, dtype=dtype)
    said = {}
    steps = [({0: 37, 2: 5}, ()), ({0: 1, 1: 130, 2: 1}, ()), ({0: 1, 2: 3, 3: 16}, ()), ({0: 20, 3: 1}, (1,)), ({1: 70, 3: 1}, (2,)), ({0: 1, 1: 1, 2: 1, 3: 1}, ())]
    for new, ended in steps:
        for r in ended:
            said.pop(r)
        ids = {r: rng.integers(0, 500, n) for r, n in new.items()}
        order, logits, nxt = m.serve_step(ids, ended)
        assert order == sorted(new)
        for r in order:
            said[r] = np.concatenate([said.get(r, np.zeros(0, np.int64)), ids[r]])
        for i, r in enumerate(order):
            want = alone(m, said[r])
            assert np.abs(logits[i] - want).max() <= REL[dtype] * np.abs(want).max(), (r, np.abs(logits[i] - want).max(), np.abs(want).max())
            assert logits[i][nxt[i]] == logits[i].max()
    assert m.serve_free() == 40 - sum(-(-len(s) // 16) for s in said.values())
    m.serve_step({}, ended=list(said))
    assert m.serve_free() == 40
    m.close()


def test_greedy_serving_repeats_generate(dev):
    m = llama(dev, positions=256)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 500, n) for n in (3, 40, 17)]
    want = [m.generate(p, 12)[len(p):] for p in prompts]
    m.cache_clear()
    m.serve_start(24, 3, page=16)
    _, _, nxt = m.serve_step(dict(enumerate(prompts)), want_logits=False)
    got = [nxt]
    for _ in range(11):
        got.append(m.serve_step({r: [got[-1][r]] for r in range(3)}, want_logits=False)[2])
    assert np.array_equal(np.array(got).T, np.array(want))
    m.close()


def test_refusals_leave_the_requests_as_they_were(dev):
    m = llama(dev, positions=100)
    with pytest.raises(nn.RuaiError, match="serve_start first"):
        m._requests = 2
        m.serve_step({0: [1]})
    for args in (dict(pages=0, requests=1), dict(pages=4, requests=0), dict(pages=4, requests=1, page=24), dict(pages=4, requests=1, dtype=7), dict(pages=4, requests=9000)):
        with pytest.raises(nn.RuaiError):
            m.serve_start(**args)
    m.serve_start(6, 3, page=16, request_pages=4)
    ids = np.arange(30)
    a = m.serve_step({0: ids})[1]
    for new, text in (({0: np.arange(80)}, "max_position"), ({0: np.arange(36)}, "exceeds its 4 pages"), ({1: np.arange(50), 2: np.arange(20)}, "more pages")):
        with pytest.raises(nn.RuaiError, match=text):
            m.serve_step(new)
    with pytest.raises(nn.RuaiError, match="token id out of range"):
        m.serve_step({1: [3, 500]})
    for new, ended in (({3: [1]}, ()), ({1: []}, ()), ({1: [1]}, (1,)), ({}, (5,))):
        with pytest.raises(ValueError):
            m.serve_step(new, ended)
    assert m.serve_free() == 4
    b = m.serve_step({0: [7], 1: ids})[1]
    assert np.abs(b[1] - a[0]).max() <= 1e-3 * np.abs(a).max()
    want = alone(m, np.concatenate([ids, [7]]))
    assert np.abs(b[0] - want).max() <= 1e-3 * np.abs(want).max()
    m.serve_stop()
    with pytest.raises(nn.RuaiError, match="serve_start first"):
        m._requests = 1
        m.serve_step({0: [1]})
    m.close()


def test_layer_lists_do_not_serve(dev):
    import zazasun_cases as zcases
    cfg = zcases.config([zcases.attention()])
    m = nn.Zazasun(dev, nn.ZazasunConfig(cfg, 0))
    for name, t in zcases.weights(cfg).items():
        m.set_tensor(name, t)
    m.build("float32")
    with pytest.raises(nn.RuaiError, match="serving over pages"):
        m.serve_start(8, 1)
    m.close()


def test_a_step_that_memory_does_not_hold_leaves_the_model_usable(dev):
    """A step whose activations take more than the device has (275 GB, refused at once) ends with an error; smaller steps, the model's own
    prompts and its decoding steps then answer as before."""
    m = llama(dev, ff=1 << 18, L=1, positions=1 << 18)
    ids, prompt = np.arange(20), np.arange(7)
    want = m.generate(prompt, 6)
    m.cache_clear()
    m.serve_start(1100, 2, page=256)
    a = m.serve_step({0: ids})[1]
    m.forward_cached(prompt[None])
    first = [m.decode_step(1) for _ in range(3)]
    with pytest.raises(nn.RuaiError, match="memory"):
        m.serve_step({1: np.zeros(1 << 18, np.int32)})
    assert m.serve_free() == 1099
    m.cache_clear()
    m.forward_cached(prompt[None])
    assert np.array_equal([m.decode_step(1) for _ in range(3)], first)
    b = m.serve_step({1: ids})[1]
    assert np.array_equal(a, b)
    m.cache_clear()
    with pytest.raises(nn.RuaiError, match="memory"):
        m.forward_cached(np.zeros((1, 1 << 18), np.int32))
    m.cache_clear()
    assert np.array_equal(m.generate(prompt, 6), want)
    m.close()


def test_models_of_one_context_serve_in_threads(dev):
    """Chunks and single tokens in f32, f16 and bf16, a model per thread, on a context whose scratch grows meanwhile: the bits of each by itself."""
    kinds = [(llama, nn.F32), (llama, nn.BF16), (MODELS["llama int4 hd 128"], nn.F16), (MODELS["llama int4 hd 128"], nn.BF16), (gpt2, nn.F32), (gpt2, nn.F16)]

    def steps(m, dtype, i):
        rng, out = np.random.default_rng(i), []
        for turn in range(6):
            m.serve_start(60, 3, page=16, dtype=dtype)
            n = 60 + 50 * turn
            for new in ({0: n, 1: 7}, {0: 1, 1: 1}, {1: 90, 2: 3}, {0: 1, 1: 1, 2: 1}):
                _, logits, nxt = m.serve_step({r: rng.integers(0, 500, t) for r, t in new.items()})
                out += [logits, nxt]
        return out

    def made(d):
        return [(make(d), dtype) for make, dtype in kinds]

    in_threads(dev, made, steps)


def in_threads(dev, made, steps):
    """The results of steps(*one, number) for each of made(device), by itself and in a thread each on a context of their own."""
    import threading
    want = []
    for i, one in enumerate(made(dev)):
        want.append(steps(*one, i))
        one[0].close()
    other = nn.Device(0)
    models, errors = made(other), []
    got, begin = [None] * len(models), threading.Barrier(len(models))

    def work(i):
        try:
            begin.wait()
            got[i] = steps(*models[i], i)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(models))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i, (a, b) in enumerate(zip(got, want)):
        assert all(np.array_equal(x, y) for x, y in zip(a, b)), i
    for m, *_ in models:
        m.close()
    nn._lib.check(other.L.ruai_ctx_destroy(other.ctx))


def test_decoding_steps_are_captured_beside_models_that_serve(dev):
    """Models that decode batches of changing sizes, each captured anew, while others serve and make the scratch grow: the bits of each by itself."""
    def steps(m, dtype, i):
        rng, out = np.random.default_rng(i), []
        for turn in range(8):
            if dtype is None:
                B = 1 + (turn + i) % 5
                m.cache_clear()
                out.append(m.forward_cached(rng.integers(0, 500, (B, 9 + 20 * turn))))
                out += [m.decode_step(B) for _ in range(12)]
            else:
                m.serve_start(60, 3, page=16, dtype=dtype)
                for new in ({0: 40 + 50 * turn, 1: 7}, {0: 1, 1: 1}, {1: 90, 2: 3}):
                    _, logits, nxt = m.serve_step({r: rng.integers(0, 500, t) for r, t in new.items()})
                    out += [logits, nxt]
        return out

    kinds = [(llama, None), (llama, nn.F32), (gpt2, None), (MODELS["llama int4 hd 128"], nn.BF16), (MODELS["llama int4 hd 128"], None), (gpt2, nn.F16)]
    in_threads(dev, lambda d: [(make(d), dtype) for make, dtype in kinds], steps)


def test_decoding_steps_are_captured_beside_tensors_that_come_and_go(dev):
    """A thread's tensors, whose blocks are set aside and waited for with the whole device, spoil no capture of another thread."""
    import threading
    m, stop, errors = llama(dev), threading.Event(), []
    x = nn.Tensor.from_numpy(dev, np.ones((4, 2048), np.float32))

    def tensors():
        try:
            while not stop.is_set():
                for n in (100, 5000, 70000):
                    kept = [nn.Tensor(dev, (n,), np.float32, nn.F32) for _ in range(40)]
                    for t in kept:
                        t.free()
                nn.Tensor.from_numpy(dev, x.numpy()).free()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    def steps():
        out = []
        for turn in range(150):
            B = 1 + turn % 5
            m.cache_clear()
            m.forward_cached(np.full((B, 3), turn % 400))
            out += [m.decode_step(B).tolist() for _ in range(2)]
        return out

    want = steps()
    others = [threading.Thread(target=tensors) for _ in range(3)]
    for t in others:
        t.start()
    try:
        got = steps()
    finally:
        stop.set()
        for t in others:
            t.join()
    assert not errors, errors
    assert got == want
    m.close()


def test_failures_of_several_threads_keep_their_texts(dev):
    """Refused calls from threads on one context: each thread reads the text of a failure, whole."""
    import threading
    import ctypes as C
    p, texts, errors = C.c_void_p(64), [], []

    def refused(page):
        try:
            for _ in range(3000):
                assert dev.L.ruai_page_plan(dev.ctx, p, p, 1, 1, page, p, 1, p, 1, p, p, p, p, p) != 0
                texts.append(dev.L.ruai_last_error(dev.ctx))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=refused, args=(8 + i * 10 ** i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert set(texts) <= {f"ruai_page_plan: pages of {8 + i * 10 ** i}: a power of two from 16 to 256".encode() for i in range(6)}
