"""GPU: penalties, biases and the allowed-token mask on logits, bit for bit the formula in f32."""
import numpy as np
import pytest
import torch

from ocelotl_b200.errors import KernelError

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_errors(backend):
    backend.take_device_errors()
    yield
    assert backend.take_device_errors() == (0, 0)


def reference(x, history=None, history_lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None,
              bias_ids=None, bias_values=None, allowed=None):
    """The formula, each step rounded to f32; history as lists of python ints a row."""
    x = x.copy()
    rows, vocab = x.shape
    with np.errstate(all="ignore"):
        for r in range(rows):
            if history is not None:
                n = min(max(int(history_lens[r]), 0), history.shape[1])
                m = min(max(0 if prompt_lens is None else int(prompt_lens[r]), 0), n)
                toks = [int(t) for t in history[r, :n]]
                seen = sorted({t for t in toks if 0 <= t < vocab})
                for t in seen:
                    if repetition is not None:
                        x[r, t] = x[r, t] / repetition[r] if x[r, t] > 0 else x[r, t] * repetition[r]
                    c = toks[m:].count(t)
                    if c and (frequency is not None or presence is not None):
                        f = np.float32(0) if frequency is None else frequency[r]
                        p = np.float32(0) if presence is None else presence[r]
                        x[r, t] = np.float32(np.float32(x[r, t] - np.float32(f * np.float32(c))) - p)
            if bias_ids is not None:
                sums = {}
                for t, b in zip(bias_ids[r], bias_values[r]):
                    if 0 <= t < vocab:
                        sums[int(t)] = np.float32(sums[int(t)] + b) if int(t) in sums else b
                for t, b in sums.items():
                    x[r, t] = np.float32(x[r, t] + b)
            if allowed is not None:
                bits = np.unpackbits(allowed[r].view(np.uint8), bitorder="little")[:vocab]
                x[r, bits == 0] = -np.inf
    return x


def run(backend, oracle, x, parts, in_place=False):
    dev = {n: torch.from_numpy(np.ascontiguousarray(t)).cuda() for n, t in parts.items()}
    rules = backend.logit_rules(**dev)
    want = reference(x, **parts)
    xd = torch.from_numpy(x).cuda()
    ids = torch.full((x.shape[0],), -9, dtype=torch.int32, device="cuda")
    out = backend.process_logits(xd, rules, out=xd if in_place else None, ids=ids)
    backend.synchronize()
    got = out.cpu().numpy()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    assert np.array_equal(got[~nan].view(np.uint32), want[~nan].view(np.uint32))
    if not in_place:
        assert np.array_equal(xd.cpu().numpy().view(np.uint32), x.view(np.uint32))
        picked = backend.greedy_sample(xd, rules=rules)
        backend.synchronize()
        assert torch.equal(picked, ids)
    assert ids.tolist() == [oracle.greedy_sample_fast(want[r]) for r in range(x.shape[0])]
    return got


def parts_of(rng, rows, vocab, n, biases=0, mask=False):
    lens = rng.integers(0, n + 1, rows).astype(np.int32)
    p = {"history": (rng.random((rows, n)) ** 3 * vocab).astype(np.int32), "history_lens": lens,
         "prompt_lens": (lens * rng.random(rows)).astype(np.int32),
         "repetition": (1 + rng.random(rows)).astype(np.float32), "frequency": rng.standard_normal(rows).astype(np.float32),
         "presence": rng.standard_normal(rows).astype(np.float32)}
    if biases:
        p["bias_ids"] = rng.integers(-1, vocab, (rows, biases)).astype(np.int32)
        p["bias_values"] = rng.standard_normal((rows, biases)).astype(np.float32)
    if mask:
        p["allowed"] = rng.integers(-2**31, 2**31, (rows, (vocab + 31) // 32)).astype(np.int32)
    return p


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4095, 4096, 4097, 32003, 128256])
@pytest.mark.parametrize("rows", [1, 5])
def test_all_rules(backend, oracle, vocab, rows):
    rng = np.random.default_rng(vocab + rows)
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 3
    run(backend, oracle, x, parts_of(rng, rows, vocab, 300, biases=70, mask=True))
    run(backend, oracle, x, parts_of(rng, rows, vocab, 1), in_place=True)


@pytest.mark.parametrize("names", [(), ("history", "history_lens", "repetition"), ("history", "history_lens", "frequency"),
                                   ("history", "history_lens", "presence", "prompt_lens"), ("history", "history_lens"),
                                   ("bias_ids", "bias_values"), ("allowed",)])
def test_each_rule_alone(backend, oracle, names):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((3, 5001)).astype(np.float32)
    p = parts_of(rng, 3, 5001, 500, biases=33, mask=True)
    run(backend, oracle, x, {n: p[n] for n in names})


def test_special_values(backend, oracle):
    rng = np.random.default_rng(8)
    vocab = 4200
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    x[0, ::3], x[1, ::5], x[2, ::2] = np.nan, np.inf, -np.inf
    x[3, 0] = np.nan
    x[4] = 0.0
    x[4, ::2] = -0.0
    p = parts_of(rng, 6, vocab, 2000, biases=40, mask=True)
    p["bias_values"][0, :5] = [np.inf, -np.inf, np.nan, 0.0, -0.0]
    p["allowed"][5] = 0  # nothing is allowed: all -inf, token 0
    p["allowed"][3] |= 1
    p["repetition"][4] = 1.0
    p["bias_ids"][3] = np.maximum(p["bias_ids"][3], 1)
    got = run(backend, oracle, x, p)
    assert np.isneginf(got[5]).all()


def test_the_same_token_often(backend, oracle):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((2, 9000)).astype(np.float32)
    p = parts_of(rng, 2, 9000, 4000, biases=300)
    p["history"][0] = 77
    p["history"][1, ::2] = 8999
    p["bias_ids"][0] = 5000
    p["bias_ids"][1, ::2] = 8999
    p["bias_ids"][1, 1::4] = 0
    run(backend, oracle, x, p)


def test_lengths_outside_the_history(backend, oracle):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((4, 700)).astype(np.float32)
    p = parts_of(rng, 4, 700, 20)
    p["history_lens"][:] = [-5, 0, 20, 9999]
    p["prompt_lens"][:] = [3, 3, -1, 9999]
    p["history"][2, 3:9] = -1  # unused places
    run(backend, oracle, x, p)


def test_ids_past_the_vocabulary_are_counted(backend, oracle):
    rng = np.random.default_rng(11)
    x = rng.standard_normal((2, 5000)).astype(np.float32)
    p = parts_of(rng, 2, 5000, 50, biases=9)
    p["history_lens"][:] = 50
    p["history"][0, 7] = 5000
    p["history"][1, 9] = 2**31 - 1
    p["bias_ids"][1, 3] = 6000
    dev = {n: torch.from_numpy(t).cuda() for n, t in p.items()}
    got = backend.process_logits(torch.from_numpy(x).cuda(), backend.logit_rules(**dev))
    backend.synchronize()
    assert backend.take_device_errors() == (3, 0)
    assert np.array_equal(got.cpu().numpy().view(np.uint32), reference(x, **p).view(np.uint32))


def test_strided_rows_of_every_alignment(backend, oracle):
    rng = np.random.default_rng(12)
    rows, vocab = 5, 4099
    p = parts_of(rng, rows, vocab, 100, biases=20, mask=True)
    wide = {n: torch.zeros(rows, t.shape[1] + 5, dtype=torch.from_numpy(t).dtype, device="cuda") for n, t in p.items()
            if t.ndim == 2}
    dev = {n: torch.from_numpy(t).cuda() for n, t in p.items()}
    for n, t in wide.items():
        t[:, 2:2 + p[n].shape[1]] = dev[n]
        dev[n] = t[:, 2:2 + p[n].shape[1]]
    rules = backend.logit_rules(**dev)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    want = reference(x, **p)
    for a in range(4):
        for b in range(4):
            src = torch.zeros(rows, vocab + 9, device="cuda")
            dst = torch.full((rows, vocab + 6), 9.0, device="cuda")
            src[:, a:a + vocab] = torch.from_numpy(x).cuda()
            backend.process_logits(src[:, a:a + vocab], rules, out=dst[:, b:b + vocab])
            backend.synchronize()
            got = dst.cpu().numpy()
            assert np.array_equal(got[:, b:b + vocab].view(np.uint32), want.view(np.uint32)), (a, b)
            assert (got[:, :b] == 9).all() and (got[:, b + vocab:] == 9).all()


def test_many_rows(backend, oracle):
    rng = np.random.default_rng(13)
    x = rng.standard_normal((300, 1500)).astype(np.float32)
    run(backend, oracle, x, parts_of(rng, 300, 1500, 64, biases=5, mask=True))


def test_captured_launch_reads_the_history_of_its_time(backend, oracle):
    rng = np.random.default_rng(14)
    x = rng.standard_normal((2, 9001)).astype(np.float32)
    p = parts_of(rng, 2, 9001, 64)
    p["history_lens"][:] = [0, 5]
    p["prompt_lens"][:] = 0
    dev = {n: torch.from_numpy(t).cuda() for n, t in p.items()}
    rules = backend.logit_rules(**dev)
    xd = torch.from_numpy(x).cuda()
    out, ids = torch.empty_like(xd), torch.empty(2, dtype=torch.int32, device="cuda")
    backend.process_logits(xd, rules, out=out, ids=ids)  # the first greedy call makes the pick's slots
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=stream):
            backend.use_current_stream()
            backend.process_logits(xd, rules, out=out, ids=ids)
    finally:
        backend.set_stream(None)
    for lens in ([0, 5], [64, 1], [3, 64]):
        p["history_lens"][:] = lens
        dev["history_lens"].copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize()
        want = reference(x, **p)
        assert np.array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))
        assert ids.tolist() == [oracle.greedy_sample_fast(w) for w in want]


def test_single_row_forms_and_no_rows(backend):
    x = torch.randn(501, device="cuda")
    rules = backend.logit_rules(allowed=torch.full((1, 16), 0, dtype=torch.int32, device="cuda"))
    assert backend.greedy_sample(x, rules=rules).tolist() == [0]
    assert int(backend.greedy_sample(x, rules=backend.logit_rules())[0]) == int(x.argmax())
    empty = backend.process_logits(torch.empty(0, 501, device="cuda"), backend.logit_rules())
    assert tuple(empty.shape) == (0, 501)


def test_refusals(backend):
    x = torch.randn(2, 100, device="cuda")
    rules = backend.logit_rules(allowed=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    f = backend.process_logits
    with pytest.raises(KernelError):
        f(x.half(), rules)
    with pytest.raises(KernelError):
        f(x.cpu(), rules)
    with pytest.raises(KernelError, match="rows"):
        f(torch.randn(3, 100, device="cuda"), rules)
    with pytest.raises(KernelError, match="words"):
        f(torch.randn(2, 129, device="cuda"), rules)
    with pytest.raises(KernelError, match="out"):
        f(x, rules, out=torch.empty(2, 99, device="cuda"))
    with pytest.raises(KernelError, match="overlaps"):
        both = torch.randn(2, 150, device="cuda")
        f(both[:, :100], rules, out=both[:, 50:])
    with pytest.raises(KernelError, match="ids"):
        f(x, rules, ids=torch.empty(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(KernelError, match="logit"):
        f(torch.empty(2, 0, device="cuda"), backend.logit_rules())
