"""Serving over the 8-bit paged cache (``mimir_b200.serving.paged``, ``Engine(kv_cache="fp8")``): the same
hidden states as the model's own cache up to the 8 bits, completions that do not depend on what
else is in the batch, forks, growth of the pool, request fields and refusals.  CPU: the PyTorch
formulations; ``-m gpu``: the kernels."""
import json
import threading
import urllib.request

import pytest
import torch

pytest.importorskip("transformers")

from mimir_b200.serving.paged import PagedDecoder, Request  # noqa: E402

VARIANTS = [dict(), dict(gates_enabled=True), dict(ngram_orders=[2, 3], ngram_buckets=97, ngram_heads=2,
                                                   ngram_contextual_gate=True),
            dict(recurrence_mode="looped")]


def _model(tmp_path, extra=None, device="cpu", dtype=torch.float32):
    from transformers import AutoModelForCausalLM
    from test_transformers_model import _export
    from mimir_b200.export.transformers_mimir2 import register
    register()
    _export(tmp_path, extra or {})
    return AutoModelForCausalLM.from_pretrained(tmp_path, dtype=dtype).to(device).eval()


class PlainBatch:
    """A :class:`mimir_b200.serving.paged.Batch` whose keys and values keep their type: the formula."""

    def __init__(self, batch, kept):
        self.batch, self.kept = batch, kept  # kept[layer, slot] -> (keys, values)
        self.slots = batch.slots

    def positions(self):
        return self.batch.positions()

    def attend(self, layer, q, k, v):
        b, out = self.batch, torch.zeros_like(q)
        pos = b.positions()
        cos, sin = b.cache.cos[pos][:, None], b.cache.sin[pos][:, None]
        half = q.shape[-1] // 2

        def turn(x):
            return x.float() * cos + torch.cat((-x[..., half:], x[..., :half]), -1).float() * sin

        q, k = turn(q), turn(k)
        start = 0
        for slot, count in zip(b.slots, b.counts):
            rows = slice(start, start + count)
            old = self.kept.get((layer, slot))
            keys, values = k[rows], v[rows].float()
            if old is not None:
                keys, values = torch.cat((old[0], keys)), torch.cat((old[1], values))
            self.kept[layer, slot] = keys, values
            group = q.shape[1] // keys.shape[1]
            s = torch.einsum("thd,jhd->htj", q[rows], keys.repeat_interleave(group, 1)) * q.shape[-1] ** -0.5
            if b.prefix_lens is None:
                seen = torch.arange(keys.shape[0], device=s.device) <= pos[rows][:, None]
                s = s.masked_fill(~seen, -torch.inf)
            out[rows] = torch.einsum("htj,jhd->thd", s.softmax(-1), values.repeat_interleave(group, 1)).to(out.dtype)
            start += count
        return out


def _teacher_forced(model, prompts, tails, plain=False):
    """Logits of the packed path for prompts and then given tokens, one at a time."""
    dec = PagedDecoder(model, page_size=16, pages=3, slots=4)
    cache, dev, slots = dec.cache, dec.device, list(range(len(prompts)))
    kept = {}

    def forward(ids, batch):
        return model.model.forward_paged(ids.to(dev), batch)

    cache.reserve(slots, [len(p) for p in prompts])
    batch = cache.batch(slots, [len(p) for p in prompts], prompts=True)
    hidden = forward(torch.tensor(sum(prompts, [])), PlainBatch(batch, kept) if plain else batch)
    out = [[x] for x in model.lm_head(hidden[batch.last_rows])]
    for s, p in zip(slots, prompts):
        dec.history[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    for t in range(len(tails[0])):
        ids = torch.tensor([tail[t] for tail in tails])
        lens = [len(p) + t + 1 for p in prompts]
        dec.history[torch.tensor(slots), torch.tensor(lens) - 1] = ids.to(dev, torch.int32)
        cache.reserve(slots, [1] * len(slots))
        batch = cache.batch(slots, [1] * len(slots))
        batch = PlainBatch(batch, kept) if plain else batch
        batch.ngram_history, batch.ngram_lens = dec.history, lens
        for row, x in zip(out, model.lm_head(forward(ids, batch))):
            row.append(x)
    return torch.stack([torch.stack(rows) for rows in out]).float()


def _both(model, vocab=96):
    """(prompts, tails, the model's own logits where they are predicted)."""
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, vocab, (n,), generator=gen).tolist() for n in (5, 1, 23)]
    tails = [torch.randint(0, vocab, (6,), generator=gen).tolist() for _ in prompts]
    full = [model(torch.tensor([p + t]).to(model.device), prefix_lengths=torch.tensor([len(p)])).logits[0, len(p) - 1:]
            for p, t in zip(prompts, tails)]
    return prompts, tails, torch.stack(full).float()


@torch.no_grad()
@pytest.mark.parametrize("extra", VARIANTS, ids=["plain", "gates", "ngram", "looped"])
def test_packed_forward_is_the_model(tmp_path, extra):
    """With keys and values as they are, the packed path gives the model's logits (float32: 12 layer calls of
    sums of at most 256 products, each rounded to 2^-24); with the 8 bits it comes near."""
    model = _model(tmp_path, extra)
    prompts, tails, full = _both(model)
    torch.testing.assert_close(_teacher_forced(model, prompts, tails, plain=True), full, atol=2e-4, rtol=2e-4)
    got = _teacher_forced(model, prompts, tails)
    assert 0 < (got - full).norm() < 0.5 * full.norm()


def test_completions_do_not_depend_on_the_batch(tmp_path):
    dec = PagedDecoder(_model(tmp_path), page_size=16, pages=1, slots=2)  # the pool and the slots have to grow
    reqs = [Request([3, 1, 4, 1, 5], max_tokens=7), Request([9] * 30, max_tokens=4, n=3),
            Request([2, 6], max_tokens=9, temperature=0.9, top_p=0.8, seed=5, n=2),
            Request([5, 3, 5], max_tokens=6, presence_penalty=1.5, frequency_penalty=0.5, repetition_penalty=1.3)]
    together = dec.generate(reqs)
    assert [len(x) for x in together] == [1, 3, 2, 1]
    assert [len(x[0]) for x in together] == [7, 4, 9, 6]
    assert together[1][0] == together[1][1] == together[1][2]  # greedy forks agree
    for r, want in zip(reqs, together):
        assert dec.generate([r])[0] == want
    assert int(dec.cache.ref_counts.sum()) == 0 and int(dec.cache.seq_lens.sum()) == 0  # all given back


def test_request_fields(tmp_path):
    dec = PagedDecoder(_model(tmp_path), slots=8)
    prompt = [7, 7, 8]
    plain = dec.generate([Request(prompt, max_tokens=8)])[0][0]
    only = dec.generate([Request(prompt, max_tokens=8, allowed_token_ids=[11, 95])])[0][0]
    assert set(only) <= {11, 95}
    assert dec.generate([Request(prompt, max_tokens=3, logit_bias={42: 1000.0})])[0][0] == [42] * 3
    banned = dec.generate([Request(prompt, max_tokens=1, logit_bias={plain[0]: -1000.0})])[0][0]
    assert banned != plain[:1]
    # a presence penalty beyond all differences forbids repetition
    once = dec.generate([Request(prompt, max_tokens=20, presence_penalty=1000.0)])[0][0]
    assert len(set(once)) == 20
    assert dec.generate([Request(prompt, max_tokens=20)], eos=plain[2])[0][0] == plain[:plain.index(plain[2]) + 1]
    for bad in (Request([], 4), Request([96], 4), Request([1] * 64, 4), Request([1], 4, n=0), Request([1], 0),
                Request([1], 4, logit_bias={96: 1.0}), Request([1], 4, allowed_token_ids=[])):
        with pytest.raises(ValueError):
            dec.generate([bad])
    assert dec.generate([Request(prompt, max_tokens=8)])[0][0] == plain
    assert len(dec.generate([Request([1] * 60, max_tokens=50)])[0][0]) == 4  # 64 positions


def _post(url, body):
    req = urllib.request.Request(url, data=json.dumps(body).encode(), headers={"Content-Type": "application/json"})
    try:
        with urllib.request.urlopen(req, timeout=60) as r:
            return r.status, r.read()
    except urllib.error.HTTPError as exc:
        return exc.code, exc.read()


def _serve(tmp_path, device, **kw):
    from test_native_serving import _tokenizer
    from mimir_b200.serving.native import Engine, make_server
    _tokenizer(tmp_path)
    engine = Engine(tmp_path, device, name="tiny", max_batch=4, batch_wait_ms=100, kv_cache="fp8", **kw)
    server = make_server(engine, "127.0.0.1", 0)
    threading.Thread(target=server.serve_forever, daemon=True).start()
    return engine, server, f"http://127.0.0.1:{server.server_address[1]}/v1/completions"


def _check_server(engine, server, url):
    try:
        bodies = [{"prompt": "w1 w2 w3", "max_tokens": 5}, {"prompt": "w4", "max_tokens": 4, "n": 3},
                  {"prompt": "w5 w6", "max_tokens": 6, "temperature": 0.7, "seed": 3},
                  {"prompt": "w7 w8", "max_tokens": 5, "logit_bias": {"10": 500}, "presence_penalty": 0.5}]
        alone = [json.loads(_post(url, b)[1]) for b in bodies]
        got = [None] * len(bodies)

        def ask(i):
            got[i] = json.loads(_post(url, bodies[i])[1])

        threads = [threading.Thread(target=ask, args=(i,)) for i in range(len(bodies))]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=120)
        for body, a, b in zip(bodies, alone, got):
            assert a["choices"] == b["choices"] and a["usage"] == b["usage"]
            assert len(a["choices"]) == body.get("n", 1) and [c["index"] for c in a["choices"]] == list(range(body.get("n", 1)))
        assert alone[1]["usage"]["completion_tokens"] <= 12 and alone[3]["choices"][0]["text"].split()[0] == "w10"
        status, raw = _post(url, bodies[0] | {"stream": True})
        lines = [x[6:] for x in raw.decode().splitlines() if x.startswith("data: ")]
        assert status == 200 and lines[-1] == "[DONE]"
        assert "".join(json.loads(x)["choices"][0]["text"] for x in lines[:-1]) == alone[0]["choices"][0]["text"]
        assert _post(url, {"prompt": "w1", "n": 0 - 1})[0] == 400
        assert _post(url, {"prompt": "w1", "repetition_penalty": -2})[0] == 400
    finally:
        server.shutdown()
        server.server_close()


def test_native_server_over_the_paged_cache(tmp_path):
    from test_transformers_model import _export
    _export(tmp_path, {})
    _check_server(*_serve(tmp_path, "cpu"))
    from mimir_b200.serving.native import Engine
    with pytest.raises(ValueError, match="model or fp8"):
        Engine(tmp_path, "cpu", kv_cache="int4")


# ---------------------------------------------------------------------------------- GPU
GPU = dict(hidden_size=256, num_heads=2, num_key_value_heads=1, max_seq_len=512)  # heads of 128


@pytest.mark.gpu
@torch.no_grad()
@pytest.mark.parametrize("extra", VARIANTS, ids=["plain", "gates", "ngram", "looped"])
def test_paged_forward_on_the_gpu(tmp_path, extra, monkeypatch):
    """The kernels are as near to the model as their PyTorch formulations on the same GPU (which round to the
    same 8 bits, and to bfloat16 in the same places)."""
    model = _model(tmp_path, GPU | extra, "cuda", torch.bfloat16)
    prompts, tails, full = _both(model)
    got = _teacher_forced(model, prompts, tails)
    monkeypatch.setenv("MIMIR_DISABLE_KERNELS", "1")
    formula = _teacher_forced(model, prompts, tails)
    assert (got - full).norm() <= 1.5 * (formula - full).norm()


@pytest.mark.gpu
def test_server_on_the_gpu(tmp_path):
    from mimir_b200.ops._ext import check_kernel_status, launch_count
    from test_transformers_model import _export
    _export(tmp_path, GPU)
    before = launch_count()
    _check_server(*_serve(tmp_path, "cuda:0", dtype=torch.bfloat16))
    assert launch_count() > before
    check_kernel_status(torch.device("cuda", 0))


@pytest.mark.gpu
def test_refusals_on_the_gpu(tmp_path):
    with pytest.raises(ValueError, match="head dimension of 128"):
        PagedDecoder(_model(tmp_path / "a", {}, "cuda", torch.bfloat16))
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        PagedDecoder(_model(tmp_path / "b", GPU, "cuda", torch.float32))


# ---------------------------------------------------------------------------------- requests that cannot be served
BAD_VALUES = [dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-40),
              dict(temperature=1.0, top_p=-1.0), dict(temperature=1.0, top_p=0.0), dict(top_p=float("nan")),
              dict(repetition_penalty=1e-40), dict(repetition_penalty=1e39), dict(repetition_penalty=float("nan")),
              dict(presence_penalty=float("nan")), dict(presence_penalty=1e39), dict(frequency_penalty=float("-inf")),
              dict(logit_bias={5: float("nan")}), dict(logit_bias={5: 1e39}), dict(temperature=1.0, seed=2 ** 70),
              dict(temperature=1.0, seed=2 ** 64 - 1, n=2), dict(temperature=1.0, seed=-2 ** 63 - 1)]


@pytest.mark.parametrize("bad", BAD_VALUES, ids=str)
def test_values_that_would_fail_in_the_batch_are_refused(bad):
    with pytest.raises(ValueError):
        Request([1, 2], **bad).check(96, 64)


@pytest.mark.parametrize("good", [dict(temperature=-1.0), dict(temperature=1e-30), dict(temperature=1.0, top_p=5.0),
                                  dict(temperature=1.0, top_p=1e-30), dict(repetition_penalty=2.0 ** -126),
                                  dict(temperature=1.0, seed=2 ** 64 - 1), dict(temperature=1.0, seed=-2 ** 63),
                                  dict(logit_bias={5: float("-inf")}, temperature=0.7), dict(presence_penalty=3e38)], ids=str)
def test_values_at_the_edges_are_served(tmp_path, good):
    dec = PagedDecoder(_model(tmp_path), slots=4)
    assert len(dec.generate([Request([1, 2], max_tokens=4, **good)])[0][0]) == 4


def test_bad_requests_do_not_reach_the_batch(tmp_path):
    from test_transformers_model import _export
    _export(tmp_path, {})
    engine, server, url = _serve(tmp_path, "cpu")
    try:
        good = {"prompt": "w1 w2", "max_tokens": 4}
        want = json.loads(_post(url, good)[1])["choices"]
        bodies = [good, {"prompt": "w3", "temperature": 1.0, "top_p": -1}, {"prompt": "w3", "temperature": 1e-39},
                  {"prompt": "w3", "temperature": 1, "seed": 2 ** 70}]
        got = [None] * len(bodies)

        def ask(i):
            got[i] = _post(url, bodies[i])

        threads = [threading.Thread(target=ask, args=(i,)) for i in range(len(bodies))]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=120)
        assert json.loads(got[0][1])["choices"] == want and [g[0] for g in got[1:]] == [400] * 3
    finally:
        server.shutdown()
        server.server_close()


def test_completions_are_bounded(tmp_path):
    """``n`` sizes slots, history and pool: one request has at most 128, and a batch of the server too."""
    with pytest.raises(ValueError, match="at most 128"):
        Request([1], n=129).check(96, 64)
    Request([1], n=128).check(96, 64)
    from test_transformers_model import _export
    _export(tmp_path, {})
    engine, server, url = _serve(tmp_path, "cpu")
    sizes, generate = [], engine.paged.generate
    engine.paged.generate = lambda requests, *a, **kw: sizes.append([r.n for r in requests]) or generate(requests, *a, **kw)
    try:
        assert _post(url, {"prompt": "w1", "n": 5000})[0] == 400
        threads = [threading.Thread(target=_post, args=(url, {"prompt": f"w{n}", "max_tokens": 1, "n": n})) for n in (60, 60, 60, 128)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=120)
        assert sorted(sum(sizes, [])) == [60, 60, 60, 128] and max(map(sum, sizes)) <= 128
        assert engine.paged.cache.page_table.shape[0] <= 128
    finally:
        server.shutdown()
        server.server_close()


def test_more_completions_than_a_call_of_the_page_operations_takes(tmp_path):
    dec = PagedDecoder(_model(tmp_path), slots=1)
    with pytest.raises(ValueError, match="4096"):
        dec.generate([Request([1], n=128)] * 33)
    assert dec.cache.page_table.shape[0] == 1


@pytest.mark.parametrize("rule", [dict(temperature=0.9, seed=1), dict()], ids=["sampled", "greedy"])
def test_a_request_without_a_token_to_choose_fails_alone(tmp_path, rule):
    """Rules that leave nothing, and logits that a poisoned cache block made NaN: that request fails, the others
    get what they get alone."""
    dec = PagedDecoder(_model(tmp_path), slots=4)
    good = Request([3, 1, 4], max_tokens=5, temperature=0.8, seed=7, n=2)
    want = dec.generate([good])[0]
    nothing = Request([2, 2], max_tokens=5, allowed_token_ids=[9], logit_bias={9: float("-inf")}, **rule)
    failed = {}
    out = dec.generate([nothing, good], failed=failed)
    assert out[1] == want and out[0] == [[]] and list(failed) == [0] and isinstance(failed[0], ValueError)
    with pytest.raises(ValueError, match="leave no token"):
        dec.generate([good, nothing])
    poisoned, failed, made = Request([5, 6], max_tokens=5, n=2, **rule), {}, {}
    for i, w, token in dec.run([poisoned, good], failed=failed):
        made.setdefault((i, w), []).append(token)
        page = int(dec.cache.page_table[1, 0])  # the second completion of the first request, while it is held
        if page >= 0:
            dec.cache.scales[0, page, 1, 0, 0] = float("nan")
    assert [made[1, 0], made[1, 1]] == want and len(made[0, 0]) == len(made[0, 1]) == 1
    assert list(failed) == [0] and isinstance(failed[0], RuntimeError)
    assert int(dec.cache.ref_counts.sum()) == 0 and int(dec.cache.seq_lens.sum()) == 0
    assert dec.generate([good])[0] == want  # the pages that were poisoned serve again


def test_the_server_answers_the_others(tmp_path):
    from test_transformers_model import _export
    _export(tmp_path, {})
    engine, server, url = _serve(tmp_path, "cpu")
    try:
        good = {"prompt": "w1 w2", "max_tokens": 4}
        want = json.loads(_post(url, good)[1])["choices"]
        bodies = [good, {"prompt": "w3", "temperature": 1.0, "allowed_token_ids": [9], "logit_bias": {"9": -1e39}}, good]
        got = [None] * len(bodies)

        def ask(i):
            got[i] = _post(url, bodies[i])

        threads = [threading.Thread(target=ask, args=(i,)) for i in range(len(bodies))]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=120)
        assert json.loads(got[0][1])["choices"] == json.loads(got[2][1])["choices"] == want and got[1][0] == 400
        engine.max_batch = 1  # one at a time
        assert _post(url, bodies[1])[0] == 400 and json.loads(_post(url, good)[1])["choices"] == want
    finally:
        server.shutdown()
        server.server_close()


def test_errors_get_a_response(tmp_path):
    """A field of a wrong type is the client's error; an engine that raises is the server's, and serves on."""
    from test_transformers_model import _export
    _export(tmp_path, {})
    engine, server, url = _serve(tmp_path, "cpu")
    try:
        good = {"prompt": "w1 w2", "max_tokens": 2}
        want = _post(url, good)
        for field in (dict(logit_bias=[5]), dict(logit_bias="5"), dict(allowed_token_ids=5), dict(n=[1]), dict(seed={})):
            assert _post(url, good | field)[0] == 400, field
        generate = engine.paged.generate

        def broken(*args):
            raise RuntimeError("out of order")

        engine.paged.generate = broken
        status, raw = _post(url, good)
        assert status == 500 and "out of order" in json.loads(raw)["error"]["message"]
        engine.paged.generate = generate
        assert json.loads(_post(url, good)[1])["choices"] == json.loads(want[1])["choices"]
    finally:
        server.shutdown()
        server.server_close()


def _raw(server, body):
    """All that the server writes for one request, as it came."""
    import socket
    data = json.dumps(body).encode()
    with socket.create_connection(server.server_address[:2], timeout=60) as s:
        s.sendall(b"POST /v1/completions HTTP/1.1\r\nHost: x\r\nConnection: close\r\nContent-Length: %d\r\n\r\n" % len(data) + data)
        out = b""
        while chunk := s.recv(65536):
            out += chunk
    return out.decode()


@pytest.mark.parametrize("kv_cache", ["fp8", "model"])
def test_a_refused_stream_has_one_status(tmp_path, kv_cache):
    """What a request's check refuses is refused before the first byte of the stream; what goes wrong later is an event."""
    from test_transformers_model import _export
    _export(tmp_path, {})
    from test_native_serving import _tokenizer
    from mimir_b200.serving.native import Engine, make_server
    _tokenizer(tmp_path)
    engine = Engine(tmp_path, "cpu", name="tiny", max_batch=4, kv_cache=kv_cache)
    server = make_server(engine, "127.0.0.1", 0)
    threading.Thread(target=server.serve_forever, daemon=True).start()
    try:
        text = _raw(server, {"prompt": "w1", "stream": True, "temperature": "warm"})
        assert text.startswith("HTTP/1.1 400 ") and text.count("HTTP/1.1") == 1 and "text/event-stream" not in text
        if kv_cache == "fp8":
            text = _raw(server, {"prompt": "w1", "stream": True, "top_p": -1})
            assert text.startswith("HTTP/1.1 400 ") and text.count("HTTP/1.1") == 1
        target = engine.paged if kv_cache == "fp8" else engine.model
        name = "run" if kv_cache == "fp8" else "generate"

        def broken(*args, **kw):
            raise ValueError("out of order")

        whole = getattr(target, name)
        setattr(target, name, broken)
        text = _raw(server, {"prompt": "w1", "stream": True})
        assert text.startswith("HTTP/1.1 200 ") and text.count("HTTP/1.1") == 1
        events = [line[6:] for line in text.splitlines() if line.startswith("data: ")]
        assert "out of order" in json.loads(events[-1])["error"]["message"]
        setattr(target, name, whole)
        assert _raw(server, {"prompt": "w1", "stream": True, "max_tokens": 3}).rstrip().endswith("data: [DONE]")
    finally:
        server.shutdown()
        server.server_close()


def test_a_stream_that_is_not_read_stops_nobody(tmp_path):
    """A reader takes one piece and no more: other requests and streams are answered; a reader that goes away ends
    its generation."""
    from test_transformers_model import _export
    _export(tmp_path, {})
    engine, server, url = _serve(tmp_path, "cpu")
    try:
        body = {"prompt": "w1 w2 w3", "max_tokens": 40, "logit_bias": {str(i): -1000 for i in range(3)}}
        ids = engine.prompt_ids(body, False)
        want = engine.complete(ids, body)
        assert want[2] == 40
        idle = engine.stream(ids, body)
        first = next(idle)[0]
        done = []
        other = threading.Thread(daemon=True, target=lambda: done.append(
            (engine.complete(ids, body), list(engine.stream(ids, body))[-1][1])))
        other.start()
        other.join(timeout=60)
        assert done == [(want, want)]
        assert first + "".join(piece for piece, _ in idle if piece is not None) == want[0]
        # a reader that goes away after its first piece
        steps, model = [], engine.model.model
        forward = model.forward_paged
        reached = threading.Event()

        def counted(*args):
            steps.append(1)
            if len(steps) == 5:
                reached.wait(30)
            return forward(*args)

        model.forward_paged = counted
        gone = engine.stream(ids, body)
        next(gone)
        gone.close()
        reached.set()
        with engine.lock:
            pass
        assert len(steps) < 40 and int(engine.paged.cache.ref_counts.sum()) == 0
    finally:
        server.shutdown()
        server.server_close()


def test_a_kernel_report_fails_the_batch(tmp_path, monkeypatch):
    """What the cache kernels report (here: a stand-in for it) is read in every step: no text comes of such a step."""
    from test_transformers_model import _export
    from mimir_b200.ops import kv_cache
    from mimir_b200.ops._ext import KernelTimeout
    _export(tmp_path, {})
    engine, server, url = _serve(tmp_path, "cpu")
    try:
        good = {"prompt": "w1 w2", "max_tokens": 4}
        want = json.loads(_post(url, good)[1])["choices"]
        codes = [0, 0, 2, 0]
        monkeypatch.setattr(kv_cache, "cache_status", lambda device: codes.pop(0) if codes else 0)
        made = []
        with pytest.raises(KernelTimeout, match="kv_cache"):
            for _, _, token in engine.paged.run([Request([1, 2], max_tokens=4)]):
                made.append(token)
        assert len(made) == 2
        codes[:] = [0, 1]
        assert _post(url, good)[0] == 500
        assert json.loads(_post(url, good)[1])["choices"] == want
        assert int(engine.paged.cache.ref_counts.sum()) == 0
    finally:
        server.shutdown()
        server.server_close()


@pytest.mark.parametrize("which", ["cache_reserve", "cache_fork"])
def test_a_pool_that_still_lacks_pages_after_growing(tmp_path, monkeypatch, which):
    """The second call's result counts as the first one's does."""
    from mimir_b200 import ops
    from mimir_b200.serving.paged import PagedCache
    cache = PagedCache(1, 2, 64, 1, 8, page_size=16, pages=4)
    cache.reserve([0], [20])
    monkeypatch.setattr(ops, which, lambda *args: torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="1 pages"):
        cache.reserve([0], [1]) if which == "cache_reserve" else cache.fork([0], [1])
    assert cache.pages.shape[1] > 4


def test_one_request_object_twice_in_a_batch(tmp_path):
    """Equal requests get equal completions, the same object or not."""
    dec = PagedDecoder(_model(tmp_path), slots=4)
    r = Request([4, 2], max_tokens=8, temperature=1.0, seed=3)
    want = dec.generate([r])[0]
    assert dec.generate([r, r]) == [want, want]


def test_one_batch_at_a_time(tmp_path):
    """A second batch beside one that is not finished would take the same slots: it is refused."""
    dec = PagedDecoder(_model(tmp_path), slots=2)
    want = dec.generate([Request([1, 2], max_tokens=6)])[0][0]
    made = dec.run([Request([1, 2], max_tokens=6)])
    tokens = [next(made)[2]]
    with pytest.raises(RuntimeError, match="not finished"):
        dec.generate([Request([3], max_tokens=2)])
    assert tokens + [t for _, _, t in made] == want
    made = dec.run([Request([1, 2], max_tokens=6)])
    next(made)
    made.close()
    assert dec.generate([Request([1, 2], max_tokens=6)])[0][0] == want


@pytest.mark.gpu
@torch.no_grad()
@pytest.mark.parametrize("rule", [dict(temperature=0.9, seed=1), dict()], ids=["sampled", "greedy"])
def test_a_request_without_a_token_to_choose_fails_alone_on_the_gpu(tmp_path, rule):
    dec = PagedDecoder(_model(tmp_path, GPU, "cuda", torch.bfloat16), slots=4)
    good = Request([3, 1, 4], max_tokens=5, temperature=0.8, seed=7, n=2)
    want = dec.generate([good])[0]
    nothing = Request([2, 2], max_tokens=5, allowed_token_ids=[9], logit_bias={9: float("-inf")}, **rule)
    poisoned, failed, lengths = Request([5, 6], max_tokens=5, **rule), {}, [0, 0, 0]
    for i, _, _ in dec.run([nothing, poisoned, good], failed=failed):
        lengths[i] += 1
        page = int(dec.cache.page_table[1, 0])
        if page >= 0:
            dec.cache.scales[0, page, 1, 0, 0] = float("nan")
    assert lengths == [0, 1, 10] and isinstance(failed[0], ValueError) and isinstance(failed[1], RuntimeError)
    assert dec.generate([good])[0] == want


@pytest.mark.gpu
@torch.no_grad()
def test_a_bad_page_fails_the_batch_on_the_gpu(tmp_path):
    from mimir_b200.ops._ext import KernelTimeout
    dec = PagedDecoder(_model(tmp_path, GPU, "cuda", torch.bfloat16), slots=2)
    want = dec.generate([Request([3, 1], max_tokens=4)])[0]
    made = dec.run([Request([3, 1], max_tokens=4)])
    next(made)
    page = int(dec.cache.page_table[0, 0])
    dec.cache.page_table[0, 0] = 10 ** 6  # skipped and reported
    with pytest.raises(KernelTimeout, match="bad page"):
        next(made)
    dec.cache.ref_counts[page] = 0
    assert dec.generate([Request([3, 1], max_tokens=4)])[0] == want


def test_no_requests_give_no_completions(tmp_path):
    assert PagedDecoder(_model(tmp_path), slots=2).generate([]) == []


def test_rules_that_float32_rounds_to_nothing(tmp_path):
    """A top_p that is zero in float32 keeps no token; a logit that a temperature takes to the edge of float32 may."""
    with pytest.raises(ValueError, match="top_p"):
        Request([1, 2], temperature=1.0, top_p=1e-320).check(96, 64)
    logits = torch.tensor([[1.0, 3.4e8, 2.0], [1.0, 1e8, 2.0]])
    reqs = [Request([1], temperature=1e-30, seed=1)] * 2
    assert PagedDecoder._sample(logits, reqs, [None, None]) == [None, 1]
