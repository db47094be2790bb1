"""Attention with a sliding window and first keys that stay visible against softmax(Q K^T / sqrt(d)) V in 64 bits."""
import pytest
import torch

from iris_b200.ops import attention as A

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of a rounding, relative


def _inputs(batch, seq, heads, kv, dtype, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed + seq + heads)
    width = (heads + 2 * kv) * 128
    qkv = torch.randn((batch * seq, width + 64), generator=g).to(device, dtype)[:, 32:32 + width]
    whole = torch.full((batch * seq + 3, heads * 128 + 16), float("nan"), dtype=dtype, device=device)
    return qkv, whole, whole[:batch * seq, 8:8 + heads * 128]


def _seen(seq, window, sinks):
    i, j = torch.arange(seq, device="cuda")[:, None], torch.arange(seq, device="cuda")
    return (j <= i) & ((j > i - window) | (j < sinks))


def _check(qkv, out, batch, seq, heads, kv, window, sinks):
    """The weights and the output are rounded to 16 bits once each: a weight by half a step of its own, which the values of the
    keys that are seen turn into at most that times their largest magnitude; ex2.approx (2 ulp), scores (129 additions in fp32
    of magnitudes of up to |q||k|, 2^-24 each) and sums are 5 % of that for bf16, and 2^-13 of it besides for fp16."""
    half, group = HALF[qkv.dtype], heads // kv
    x = qkv.double().view(batch, seq, heads + 2 * kv, 128)
    seen = _seen(seq, window, sinks)
    for b in range(batch):
        for h in range(heads):
            q, k, v = x[b, :, h], x[b, :, heads + h // group], x[b, :, heads + kv + h // group]
            s = (q @ k.T / 128 ** 0.5).masked_fill(~seen, float("-inf"))
            ref = torch.softmax(s, 1) @ v
            v_max = torch.stack([v[seen[i]].abs().max() for i in range(seq)]) if seq <= 200 else v.abs().max().expand(seq)
            tol = half * ref.abs() + ((1.05 * half + 2.0 ** -13) * v_max)[:, None]
            err = (out.unflatten(0, (batch, seq)).unflatten(2, (heads, 128))[b, :, h].double() - ref).abs()
            assert bool((err <= tol).all()), f"batch {b} head {h}: {(err / tol).max().item()} of the tolerance"


def _run(batch, seq, heads, kv, window, sinks, dtype):
    qkv, whole, out = _inputs(batch, seq, heads, kv, dtype)
    status = torch.zeros(16, dtype=torch.int32, device="cuda")
    A.attention_window_fwd(qkv, out, batch, seq, heads, kv, window=window, sinks=sinks, status=status)
    torch.cuda.synchronize()
    assert int(status[0]) == 0, f"a wait of the kernel ran out: {status[:8].tolist()}"
    rest = whole.clone()
    rest[:batch * seq, 8:8 + heads * 128] = float("nan")
    assert bool(torch.isnan(rest.float()).all()), "wrote outside the output"
    return qkv, out


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seq", [1, 2, 77, 127, 128, 129, 256, 300, 640])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (33, 0), (128, 4), (129, 130), (200, 300), (5000, 0)])
def test_lengths_and_windows(seq, window, sinks, dtype):
    """Few heads: the keys of a tile of queries are shared out."""
    _check(*_run(2, seq, 3, 1, window, sinks, dtype), 2, seq, 3, 1, window, sinks)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,seq,heads,kv", [(3, 640, 40, 40), (2, 1000, 40, 8), (1, 1300, 64, 2), (9, 129, 80, 80), (70, 77, 10, 5)])
@pytest.mark.parametrize("window,sinks", [(100, 0), (256, 4), (300, 200), (9999, 0)])
def test_many_heads(batch, seq, heads, kv, window, sinks, dtype):
    """Pairs of query tiles, several items per CTA, an odd number of tiles, grouped heads."""
    qkv, out = _run(batch, seq, heads, kv, window, sinks, dtype)
    x, o = qkv.view(batch, seq, -1), out.view(batch, seq, -1)
    for b in {0, batch - 1}:
        for h in {0, heads // 2, heads - 1}:                # one head at a time
            g = h // (heads // kv)
            part = torch.cat([x[b, :, n * 128:(n + 1) * 128] for n in (h, heads + g, heads + kv + g)], 1)
            _check(part, o[b, :, h * 128:(h + 1) * 128], 1, seq, 1, 1, window, sinks)


@gpu
@pytest.mark.parametrize("batch,seq,heads", [(1, 512, 2), (2, 1024, 40)])
def test_a_window_of_all_keys_is_causal_attention(batch, seq, heads):
    """Both are within the bounds of the same formula.  (Not bit by bit: the weights of the two are scaled by different powers of
    e before they are rounded, as far apart as 2^8, since the windowed form renews a row's maximum less often.)"""
    qkv, _, out = _inputs(batch, seq, heads, heads, torch.bfloat16)
    want = torch.empty_like(out)
    A.attention_fwd(qkv, want, batch, seq, heads)
    A.attention_window_fwd(qkv, out, batch, seq, heads, window=seq)
    w = heads * 128
    for b in range(batch):
        for h in {0, heads - 1}:
            x = qkv[b * seq:(b + 1) * seq]
            part = torch.cat([x[:, n * w + h * 128:n * w + (h + 1) * 128] for n in range(3)], 1)
            for o in (out, want):
                _check(part, o[b * seq:(b + 1) * seq, h * 128:(h + 1) * 128], 1, seq, 1, 1, seq, 0)


@gpu
@pytest.mark.parametrize("batch,heads", [(1, 2), (2, 60)])   # keys of a query tile shared out; pairs of query tiles
def test_hidden_keys_weigh_nothing(batch, heads):
    """Keys and values that a query does not see reach it with no bit, whatever finite size they have; neither does the next
    sequence, NaN and all."""
    seq, window, sinks = 500, 70, 5
    qkv, _, out = _inputs(batch, seq, heads, heads, torch.bfloat16)
    A.attention_window_fwd(qkv, out, batch, seq, heads, window=window, sinks=sinks)
    w = heads * 128
    other, got = qkv.clone(), torch.empty_like(out)
    x = other.view(batch, seq, 3 * w)
    x[0, 100:130, 2 * w:] = 3.0e38
    x[0, 100:130, w:2 * w] *= -50.0
    if batch > 1:
        x[1] = float("nan")
    A.attention_window_fwd(other, got, batch, seq, heads, window=window, sinks=sinks)
    a, b = (t.view(batch, seq, w)[0] for t in (out, got))
    assert torch.equal(a[:100], b[:100]) and torch.equal(a[199:], b[199:])
    assert not torch.equal(a[129:199], b[129:199])


@gpu
@pytest.mark.parametrize("batch,heads", [(1, 1), (2, 80)])
def test_nan_of_a_key_reaches_the_queries_that_see_it(batch, heads):
    seq, window, sinks, w = 400, 90, 3, heads * 128
    for key, rows in ((200, list(range(200, 290))), (1, list(range(1, 400)))):
        qkv, _, out = _inputs(batch, seq, heads, heads, torch.bfloat16)
        qkv[key, w:w + 128] = float("nan")
        A.attention_window_fwd(qkv, out, batch, seq, heads, window=window, sinks=sinks)
        nan = torch.isnan(out.float())
        want = torch.zeros_like(nan)
        want[rows, :128] = True
        assert torch.equal(nan, want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [1, 40])                  # keys of a query tile shared out; pairs of query tiles
@pytest.mark.parametrize("first", [0, 4000])                # among the first keys; a key of the window
def test_weights_far_below_the_largest_count(first, heads, dtype):
    """One key takes nearly all of a row's weight and has values of zero; 8190 others of weight exp(-18) = 2^-25.97 each make up the
    output.  A weight is off by half a step of its 16 bits (bf16 2^-8; fp16 as much as 2^-7 where it is that far below the largest,
    since it has a number of its own down to 2^-32 of the row's maximum), ex2, scores and sums by less than 2^-10 together."""
    seq = 8192
    qkv, _, out = _inputs(1, seq, heads, heads, dtype)
    x = qkv.unflatten(1, (3, heads, 128))
    x[:, :2] = 0.0
    x[:, 0, :, 0] = 128 ** 0.5
    x[:, 0, :, 1] = 0.0
    x[:, 2] = 1.0
    x[first, 1, :, 0] = 18.0
    x[first, 2] = 0.0
    A.attention_window_fwd(qkv, out, 1, seq, heads, window=5000, sinks=1)
    score = float(x[0, 0, 0, 0].double()) * 18.0 / 128 ** 0.5           # (the root of 128 is rounded too)
    for row in (4500, 8191):
        n = min(row + 1, 5000) + (1 if row >= 5000 else 0)              # keys that the row sees
        others = (n - 1) * torch.tensor(-score, dtype=torch.float64).exp().item()
        want = others / (1 + others)
        rel = HALF[dtype] + 2.0 ** -7 + 2.0 ** -10
        got = out[row].double()
        assert bool(((got - want).abs() <= rel * want).all()), (row, got[0].item(), want)


@gpu
@pytest.mark.parametrize("heads", [1, 40])                  # keys of a query tile shared out; pairs of query tiles
@pytest.mark.parametrize("sign", [1, -1])
def test_huge_scores_stay_finite(sign, heads):
    """fp16, scores of up to 2^27 (in powers of two) of either sign, each off by as much as 4: every 50th key is far above the
    others, so that the values of the largest one that a row sees are its output, to the rounding of its weight and its own."""
    seq, window = 900, 130
    qkv, _, out = _inputs(1, seq, heads, heads, torch.float16)
    x = qkv.unflatten(1, (3, heads, 128))
    g = torch.Generator().manual_seed(3)
    size = torch.randint(20, 50, (seq // 50,), generator=g).unique().flip(0).repeat(18)[:18] * 600.0
    x[:, :2] = 0.0
    x[:, 0, :, 0] = 20000.0
    x[:, 1, :, 0] = 3000.0 if sign > 0 else -60000.0
    x[::50, 1, :, 0] = (size if sign > 0 else size - 59000.0)[:, None].to("cuda", torch.float16)
    A.attention_window_fwd(qkv, out, 1, seq, heads, window=window)
    k, v = x[:, 1, 0, 0].double(), x[:, 2].double()
    for row in range(0, seq, 7):
        seen = torch.arange(max(0, row - window + 1), row + 1, device="cuda")
        best = k[seen] == k[seen].max()
        if best.sum() > 1:                                   # (rows that see none of the large ones, or two alike)
            continue
        want = v[seen[best]][0].flatten()
        assert bool(((out[row].double() - want).abs() <= 2 * HALF[torch.float16] * want.abs() + 2.0 ** -24).all()), row


@gpu
def test_in_a_graph_and_on_another_stream():
    qkv, _, out = _inputs(2, 300, 4, 2, torch.bfloat16)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    A.attention_window_fwd(qkv, out, 2, 300, 4, 2, window=50, stream=st.cuda_stream)
    torch.cuda.synchronize()
    first = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.attention_window_fwd(qkv, out, 2, 300, 4, 2, window=50)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    qkv.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    _check(qkv, out, 2, 300, 4, 2, 50, 0)


@gpu
@pytest.mark.parametrize("batch,seq,heads,kv", [(2, 300, 4, 2), (3, 640, 40, 8)])
def test_output_over_the_queries(batch, seq, heads, kv):
    qkv, _, out = _inputs(batch, seq, heads, kv, torch.bfloat16)
    A.attention_window_fwd(qkv, out, batch, seq, heads, kv, window=100, sinks=2)
    over = qkv[:, :heads * 128]
    A.attention_window_fwd(qkv, over, batch, seq, heads, kv, window=100, sinks=2)
    assert torch.equal(over, out)


@gpu
def test_offsets_beyond_32_bits():
    """A matrix of more than 2^31 elements: the last rows of the last head are those of a short matrix with the same keys."""
    seq, heads, window = 180000, 32, 100
    width = 3 * heads * 128
    qkv = torch.zeros((seq, width), dtype=torch.bfloat16, device="cuda")
    assert qkv.numel() > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    tail = torch.randn((256, width), generator=g, device="cuda").to(torch.bfloat16)
    qkv[-256:] = tail
    out = torch.empty((seq, heads * 128), dtype=torch.bfloat16, device="cuda")
    A.attention_window_fwd(qkv, out, 1, seq, heads, window=window)
    for h in (0, heads - 1):
        part = torch.cat([tail[:, (n * heads + h) * 128:(n * heads + h + 1) * 128] for n in range(3)], 1)
        ref = torch.empty((256, 128), dtype=torch.bfloat16, device="cuda")
        A.attention_window_fwd(part, ref, 1, 256, 1, window=window)
        # of the same keys, but grouped into other tiles: each is within the bounds of _check, the values' maximum times 2^-7
        got = out[-256:, h * 128:(h + 1) * 128]
        bound = 2 * 1.05 * 2.0 ** -7 * tail[:, 2 * heads * 128:].abs().max().item()
        assert (got[window:].float() - ref[window:].float()).abs().max().item() <= bound


@gpu
@pytest.mark.parametrize("batch,seq,heads,kv", [(2, 300, 4, 2), (3, 640, 40, 8)])
def test_waits_that_may_run_out(batch, seq, heads, kv):
    """A limit of a microsecond: the call comes back, with or without having recorded that a wait ran out, with nothing left on its
    way, and the next one is right."""
    qkv, _, out = _inputs(batch, seq, heads, kv, torch.bfloat16)
    status = torch.zeros(64, dtype=torch.int32, device="cuda")
    for _ in range(20):
        A.attention_window_fwd(qkv, out, batch, seq, heads, kv, window=100, timeout_ms=1e-3, status=status)
    torch.cuda.synchronize()
    assert status[0].item() in (0, 1), status[:8]
    A.attention_window_fwd(qkv, out, batch, seq, heads, kv, window=100)
    _check(qkv, out, batch, seq, heads, kv, 100, 0)


@gpu
def test_no_rows():
    qkv, _, out = _inputs(1, 4, 2, 1, torch.bfloat16)
    assert A.attention_window_fwd(qkv[:0], out[:0], 0, 4, 2, 1, window=4).shape == (0, 256)


def test_refusals():
    qkv, _, out = _inputs(2, 10, 4, 2, torch.bfloat16, device="cpu")
    ok = dict(qkv=qkv, out=out, batch=2, seq=10, heads=4, kv_heads=2, window=4)
    with pytest.raises(TypeError):
        A.attention_window_fwd(**{**ok, "out": out.half()})
    for bad in (dict(kv_heads=3), dict(kv_heads=0), dict(kv_heads=4), dict(seq=9), dict(batch=3), dict(window=0), dict(window=-1),
                dict(sinks=-1), dict(qkv=qkv.t().contiguous().t()), dict(out=out[:, :128]), dict(qkv=qkv[None])):
        with pytest.raises(ValueError):
            A.attention_window_fwd(**{**ok, **bad})
    wide = torch.zeros((20, 2000), dtype=torch.bfloat16)
    for bad in (wide[:, 512:1024], wide[:, 800:1312], wide[:1, :512].expand(20, -1)):      # over the keys; over the values; one row
        with pytest.raises(ValueError, match="overlap"):
            A.attention_window_fwd(**{**ok, "qkv": wide[:, :1024], "out": bad})
    tall = torch.zeros((21, 1024), dtype=torch.bfloat16)                                 # the queries of the next token
    with pytest.raises(ValueError, match="overlap"):
        A.attention_window_fwd(**{**ok, "qkv": tall[:20], "out": tall[1:, :512]})
    for fine in (out, wide[:, :512], wide[:, 1024:1536]):                                # of its own; the queries; beside them
        with pytest.raises(ValueError, match="CUDA device"):
            A.attention_window_fwd(**{**ok, "qkv": wide[:, :1024], "out": fine})


def test_one_token_over_its_queries_whatever_its_strides():
    """Along one row a stride says nothing."""
    qkv, _, _ = _inputs(1, 1, 4, 2, torch.bfloat16, device="cpu")
    with pytest.raises(ValueError, match="CUDA device"):
        A.attention_window_fwd(qkv, torch.as_strided(qkv, (1, 512), (0, 1)), 1, 1, 4, 2, window=4)


def test_a_status_that_is_no_block_is_refused():
    """A record has 32 bytes; what is smaller, strided or misaligned would be written past."""
    qkv, _, out = _inputs(2, 10, 4, 2, torch.bfloat16, device="cpu")
    memory = torch.zeros(17, dtype=torch.int32)
    for bad in (memory[:1], memory[:7], memory[1:], memory[::2][:8]):
        with pytest.raises(ValueError, match="status"):
            A.attention_window_fwd(qkv, out, 2, 10, 4, 2, window=4, status=bad)
    with pytest.raises(ValueError, match="CUDA device"):
        A.attention_window_fwd(qkv, out, 2, 10, 4, 2, window=4, status=memory[:8])


@gpu
def test_refusals_of_the_native_entry():
    wide = torch.zeros((20, 2000), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="16-byte"):
        A.attention_window_fwd(wide[:, 1:1025], wide[:, 1200:1712], 2, 10, 4, 2, window=4)
    with pytest.raises(RuntimeError, match="16-byte"):
        A.attention_window_fwd(wide[:1].expand(20, -1)[:, :1024], wide[:, 1200:1712], 2, 10, 4, 2, window=4)
