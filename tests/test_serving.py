"""The decoder with positions, head norms, grouped heads and windows against the unsharded fp32 oracle: whole sequences, and the
same sequences as prompts followed by single tokens over a paged cache."""
import pytest
import torch

import iris_b200 as iris
from iris_b200.models.tp_block import TPConfig, TPDecoder, TPDecoderBaseline, reference_forward

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

SIZES = dict(hidden=512, n_heads=4, head_dim=128, intermediate=1024, n_layers=2, seed=4)
KINDS = {
    "plain": dict(),
    "grouped": dict(n_kv_heads=2, rope_theta=10000.0, qk_norm=True),
    "window": dict(rope_theta=10000.0, window=50, sinks=3),
    "part": dict(n_kv_heads=2, rope_theta=10000.0, rotary_dim=32, interleaved=True, window=9),
}


def _inputs(batch, seq, hidden=512):
    g = torch.Generator(device="cuda").manual_seed(batch + seq)
    return torch.randn((batch, seq, hidden), generator=g, device="cuda").to(torch.bfloat16)


def _near(got, ref):
    """Bounds of tests/test_gpu_tp_block.py for the same depth and width."""
    err = (got.float() - ref).abs()
    assert err.mean().item() < 2e-2 and err.max().item() < 0.25, (err.mean().item(), err.max().item())


@pytest.mark.parametrize("world", [1, 2])
@pytest.mark.parametrize("kind", ["grouped", "window", "part"])
def test_whole_sequences(kind, world):
    batch, seq = 4, 192 if kind != "grouped" else 256      # (with peers, a rank has a multiple of 128 rows)
    cfg = TPConfig(batch=batch, seq=seq, **SIZES, **KINDS[kind])
    ranks = iris.Iris.local_world(world, heap_size=192 << 20)
    model = TPDecoder(ranks, cfg)
    x = _inputs(batch, seq).view(batch * seq, -1)
    ts = cfg.tokens // world
    shards = [x[r * ts:(r + 1) * ts].clone() for r in range(world)]
    model.forward(shards)
    model.check()
    _near(torch.cat(shards, 0), reference_forward(x, cfg))
    model.close()
    ranks[0].close()


@pytest.mark.parametrize("world,kind,batch,seq,steps", [
    (1, "plain", 4, 96, 40), (1, "grouped", 4, 96, 40), (1, "window", 4, 96, 40), (1, "part", 5, 77, 40), (2, "grouped", 256, 8, 30)])
@pytest.mark.parametrize("graph", [False, True])
def test_prompts_then_single_tokens(kind, world, batch, seq, steps, graph):
    """Prompts of several lengths, one of them empty, then tokens one by one, a request that pauses, one that ends and whose
    pages another gets: every row is the oracle's for the whole sequence."""
    more = dict(SIZES, **KINDS[kind], positions=seq + steps)
    pre, one = TPConfig(batch=batch, seq=seq, **more), TPConfig(batch=batch, seq=1, **more)
    whole = TPConfig(batch=batch, seq=seq + steps, **more)
    ranks = iris.Iris.local_world(world, heap_size=192 << 20)
    prefill = TPDecoder(ranks, pre)
    decode = TPDecoder(ranks, one, weights=prefill)
    cache = prefill.make_cache(pages=batch * -(-(seq + steps) // 16), page_size=16, max_batch=batch, max_len=seq + steps)
    x = _inputs(batch, seq + steps)
    want = reference_forward(x.view(-1, 512), whole).view(batch, seq + steps, 512)
    lens = [(seq, 17, 0, 50)[b % 4] % (seq + 1) for b in range(batch)]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731

    def run(model, rows, new):
        n = rows.shape[0] // world
        shards = [rows[r * n:(r + 1) * n].clone() for r in range(world)]
        model.forward(shards, cache=cache, new_lens=new)
        model.check()
        return torch.cat(shards, 0)
    got = run(prefill, x[:, :seq].reshape(-1, 512), ints(lens)).view(batch, seq, 512)
    real = torch.arange(seq) < torch.tensor(lens)[:, None]
    _near(got[real], want[:, :seq][real])
    new = ints([1] * batch)
    per = batch // world
    shards = [torch.empty((per, 512), dtype=torch.bfloat16, device="cuda") for _ in range(world)]
    recorded = None
    if graph:
        before = [c.lens.clone() for c in cache], [c.free_count.clone() for c in cache], [c.block_table.clone() for c in cache]
        for s in shards:
            s.zero_()
        recorded = decode.capture(shards, cache=cache, new_lens=new)
        assert all(torch.equal(c.lens, l) and torch.equal(c.free_count, f) and torch.equal(c.block_table, t)
                   for c, l, f, t in zip(cache, *before))
    for step in range(steps):
        active = [not (b % 4 == 1 and step % 5 == 2) for b in range(batch)]
        if step == 20:                                            # request 3 ends, and begins again from its first token
            for c in cache:
                c.release(ints([int(b % 4 == 3) for b in range(batch)]))
            lens = [0 if b % 4 == 3 else n for b, n in enumerate(lens)]
        new.copy_(ints([int(a) for a in active]))
        rows = x[torch.arange(batch), lens]
        if graph:
            for r, s in enumerate(shards):
                s.copy_(rows[r * per:(r + 1) * per])
            recorded.replay()
            decode.check()
            out = torch.cat(shards, 0)
        else:
            out = run(decode, rows, new)
        _near(out[active], want[torch.arange(batch), lens][active])
        lens = [n + a for n, a in zip(lens, active)]
    assert all(c.lens.tolist() == lens for c in cache)
    decode.close(), prefill.close()
    ranks[0].close()


def _forward(model, rows, cache, new):
    shards = [rows.clone()]
    model.forward(shards, cache=cache, new_lens=torch.tensor(new, dtype=torch.int32, device="cuda"))
    model.check()
    return shards[0]


def test_a_request_stops_at_the_caches_longest_length():
    """Angles for 71 positions, a cache of requests of up to 71 tokens, pages of 16: the 72nd token is not taken, and its request
    answers as before, whoever had the rest of its page earlier."""
    more = dict(SIZES, **KINDS["grouped"], positions=71)
    ctx = iris.iris(192 << 20)
    prefill = TPDecoder(ctx, TPConfig(batch=2, seq=70, **more))
    decode = TPDecoder(ctx, TPConfig(batch=2, seq=1, **more), weights=prefill)
    cache = prefill.make_cache(10, 16, 2, 71)
    x = _inputs(2, 71)
    want = reference_forward(x.view(142, -1), TPConfig(batch=2, seq=71, **more)).view(2, 71, -1)
    _forward(prefill, x[:, :70].reshape(140, -1), cache, [70, 70])
    _near(_forward(decode, x[:, 70].contiguous(), cache, [1, 1]), want[:, 70])
    for _ in range(3):
        _forward(decode, x[:, 70].contiguous(), cache, [1, 1])              # (and check() finds nothing recorded)
        assert cache[0].lens.tolist() == [71, 71] and decode.cache_positions.tolist() == [-1, -1]
    prefill.close(), decode.close(), ctx.close()


@pytest.mark.parametrize("kind", ["plain", "grouped", "window"])
def test_a_prompt_for_a_request_that_holds_tokens_gets_nothing(kind):
    """A prompt attends over its own rows alone, so a request that goes on takes single tokens; others in the call are served."""
    more = dict(SIZES, **KINDS[kind], positions=64)
    ctx = iris.iris(192 << 20)
    prefill = TPDecoder(ctx, TPConfig(batch=2, seq=40, **more))
    decode = TPDecoder(ctx, TPConfig(batch=2, seq=1, **more), weights=prefill)
    cache = prefill.make_cache(16, 16, 2, 64)
    x = _inputs(2, 40)
    want = reference_forward(x.view(80, -1), TPConfig(batch=2, seq=40, **more)).view(2, 40, -1)
    got = _forward(prefill, x.view(80, -1), cache, [12, 0]).view(2, 40, -1)
    _near(got[0, :12], want[0, :12])
    free = cache[0].free_count.item()
    got = _forward(prefill, x.view(80, -1), cache, [9, 30]).view(2, 40, -1)
    assert cache[0].lens.tolist() == [12, 30] and cache[0].free_count.item() == free - 2
    _near(got[1, :30], want[1, :30])
    _near(_forward(decode, x[torch.arange(2), [12, 30]], cache, [1, 1]), want[torch.arange(2), [12, 30]])
    prefill.close(), decode.close(), ctx.close()


@pytest.mark.parametrize("kind,seq,attention", [
    ("plain", 128, "iris"), ("plain", 96, "iris"), ("grouped", 96, "iris"), ("window", 128, "iris"), ("plain", 128, "sdpa")])
@pytest.mark.parametrize("rubbish", [float("nan"), float("inf"), 3.0e38])
def test_rows_of_no_token_reach_nothing(kind, seq, attention, rubbish):
    """A prompt's padding may hold anything, NaN and infinity too."""
    more = dict(SIZES, **KINDS[kind], positions=seq)
    cfg = TPConfig(batch=3, seq=seq, **more)
    ctx = iris.iris(192 << 20)
    prefill = TPDecoder(ctx, cfg, attention=attention)
    decode = TPDecoder(ctx, TPConfig(batch=3, seq=1, **more), weights=prefill)
    cache = prefill.make_cache(3 * 8, 16, 3, seq)
    x, lens = _inputs(3, seq), [seq - 30, 1, 0]
    want = reference_forward(x.view(3 * seq, -1), cfg).view(3, seq, -1)
    padded = x.clone()
    for b, n in enumerate(lens):
        padded[b, n:] = rubbish
    got = _forward(prefill, padded.view(3 * seq, -1), cache, lens).view(3, seq, -1)
    for b, n in enumerate(lens):
        if n:
            _near(got[b, :n], want[b, :n])
    step = x[torch.arange(3), lens].clone()
    step[1] = rubbish                                                       # no token either
    got = _forward(decode, step, cache, [1, 0, 1])
    _near(got[[0, 2]], want[torch.arange(3), lens][[0, 2]])
    prefill.close(), decode.close(), ctx.close()


@pytest.mark.parametrize("kind", [dict(rope_theta=10000.0), dict(qk_norm=True), dict()])
@pytest.mark.parametrize("with_cache", [False, True])
def test_the_librarys_attention_where_it_is_asked_for(kind, with_cache, monkeypatch):
    """``attention="sdpa"`` goes for configurations with positions or head norms and for calls with a cache too, at any length."""
    from iris_b200.ops import attention as A
    cfg = TPConfig(batch=2, seq=96, **SIZES, **kind)
    ctx = iris.iris(192 << 20)
    model = TPDecoder(ctx, cfg, attention="sdpa")
    x = _inputs(2, 96).view(192, -1)

    def never(*a, **k):
        raise AssertionError("the own kernel was called")
    monkeypatch.setattr(A, "attention_window_fwd", never)
    monkeypatch.setattr(A, "attention_fwd", never)
    shards = [x.clone()]
    if with_cache:
        got = _forward(model, x, model.make_cache(12, 16, 2, 96), [96, 96])
    else:
        model.forward(shards)
        got = shards[0]
    model.check()
    _near(got, reference_forward(x, cfg))
    model.close(), ctx.close()


def test_heads_that_cannot_be_decoded_are_refused_before_pages_are_taken():
    more = dict(SIZES, hidden=512, rope_theta=10000.0, positions=40)
    more.update(n_heads=16, head_dim=32)
    ctx = iris.iris(192 << 20)
    prefill = TPDecoder(ctx, TPConfig(batch=2, seq=32, **more))
    decode = TPDecoder(ctx, TPConfig(batch=2, seq=1, **more), weights=prefill)
    cache = prefill.make_cache(8, 16, 2, 40)
    _forward(prefill, _inputs(2, 32).view(64, -1), cache, [20, 3])
    with pytest.raises(ValueError, match="64, 128 or 256"):
        _forward(decode, _inputs(2, 1).view(2, -1), cache, [1, 1])
    assert cache[0].lens.tolist() == [20, 3] and cache[0].free_count.item() == 5
    prefill.close(), decode.close(), ctx.close()


def test_captured_prompts():
    """Prompts recorded once and replayed with other rows and lengths: requests that hold tokens and padding of NaN included."""
    more = dict(SIZES, **KINDS["window"], positions=64)
    ctx = iris.iris(192 << 20)
    prefill = TPDecoder(ctx, TPConfig(batch=3, seq=40, **more))
    cache = prefill.make_cache(9, 16, 3, 64)
    x = _inputs(3, 40)
    want = reference_forward(x.view(120, -1), TPConfig(batch=3, seq=40, **more)).view(3, 40, -1)
    rows, new = torch.empty((120, 512), dtype=torch.bfloat16, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    graph = prefill.capture([rows], cache=cache, new_lens=new)
    held = [0, 0, 0]
    for lens in ([40, 3, 0], [5, 0, 20], [0, 0, 1], [12, 33, 0]):
        padded = x.clone()
        for b, n in enumerate(lens):
            padded[b, n:] = float("nan")
        rows.copy_(padded.view(120, -1))
        new.copy_(torch.tensor(lens))
        graph.replay()
        prefill.check()
        given = [b for b in range(3) if lens[b] and not held[b]]
        held = [lens[b] if b in given else held[b] for b in range(3)]
        assert cache[0].lens.tolist() == held
        for b in given:
            _near(rows.view(3, 40, -1)[b, :lens[b]], want[b, :lens[b]])
        if lens[2] == 1:
            cache[0].release(torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda"))
            held[:2] = [0, 0]
    prefill.close(), ctx.close()


def test_refusals():
    ctx = iris.iris(192 << 20)
    cfg = TPConfig(batch=2, seq=64, **SIZES, **KINDS["grouped"])
    model = TPDecoder(ctx, cfg)
    x = [torch.zeros((128, 512), dtype=torch.bfloat16, device="cuda")]
    new = torch.ones(2, dtype=torch.int32, device="cuda")
    for bad in (dict(new_lens=new), dict(cache=model.make_cache(4, 16, 2, 64)), dict(cache=model.make_cache(4, 16, 3, 64), new_lens=new),
                dict(cache=model.make_cache(4, 16, 2, 65), new_lens=new), dict(cache=[], new_lens=new)):
        with pytest.raises(ValueError):
            model.forward(x, **bad)
    with pytest.raises(ValueError):
        TPDecoder(ctx, TPConfig(batch=2, seq=64, **SIZES, n_kv_heads=3))
    with pytest.raises(ValueError):
        TPDecoder(ctx, TPConfig(batch=2, seq=64, **SIZES, window=8), attention="sdpa")
    with pytest.raises(ValueError):
        TPDecoder(ctx, TPConfig(batch=2, seq=64, **SIZES), weights=model)
    with pytest.raises(ValueError):
        TPDecoderBaseline(cfg, 0, 1, "cuda")
    model.close(), ctx.close()


def test_example_decodes():
    """The example runs its prompts and tokens and agrees with the oracle."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    args = ("--hidden 512 --heads 4 --kv_heads 2 --intermediate 1024 --layers 2 --batch 2 --seq 60 --decode 5 --rope_theta 10000 "
            "--qk_norm --window 30 --sinks 2 -v --heap_size 268435456").split()
    run = subprocess.run([sys.executable, os.path.join(root, "examples", "10_tp_block", "tp_block.py"), *args], capture_output=True,
                         text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "us a step" in run.stdout
