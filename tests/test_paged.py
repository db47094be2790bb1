"""The paged cache's operators against plain implementations in 64 bits: attention of one new token, pages taken and given
back, and the refusals of both."""
import ctypes
import math
import random

import pytest
import torch

from iris_b200 import _native
from iris_b200.ops import paged as P

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of a rounding, relative


def _visible(n, window, sinks):
    start = max(0, n - window) if window else 0
    return list(range(min(sinks, start))) + list(range(start, n))


class Case:
    """A cache in which everything that no query sees is NaN, tables with rubbish behind the last page, and strided queries."""

    def __init__(self, lens, heads, kv, dim, page, dtype, window=0, sinks=0, order="page_slot", wide=None, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed + 7 * len(lens) + dim)
        rng = random.Random(seed)
        self.lens, self.window, self.sinks, self.page, self.kv = lens, window, sinks, page, kv
        wide = wide or max(1, max(math.ceil(n / page) for n in lens))
        pages = sum(math.ceil(n / page) for n in lens) + 2
        ids = list(range(pages))
        rng.shuffle(ids)
        table = torch.full((len(lens), wide + 3), 0x7ffffff0, dtype=torch.int32)   # three columns of another matrix behind
        data = torch.full((2, pages, page, kv, dim), float("nan"))
        for b, n in enumerate(lens):
            for i in range(math.ceil(n / page)):
                table[b, i] = ids.pop()
            for j in _visible(n, window, sinks):
                data[:, table[b, j // page], j % page] = torch.randn((2, kv, dim), generator=g)
        both = torch.randn((len(lens), heads + 2, dim + 16), generator=g)
        if order == "page_head":
            data = data.transpose(2, 3).contiguous().to(device, dtype).transpose(2, 3)
        else:
            data = data.to(device, dtype)
        self.k, self.v = data[0], data[1]
        self.q = both.to(device, dtype)[:, 1:heads + 1, 8:dim + 8]
        self.table = table.to(device)[:, :wide]
        self.len_t = torch.tensor(lens, dtype=torch.int32, device=device)
        self.whole = torch.full((len(lens), heads + 1, dim + 8), float("nan"), dtype=dtype, device=device)
        self.out = self.whole[:, :heads, :dim]
        self.lse = torch.full((len(lens), heads + 5), float("nan"), device=device)[:, :heads]

    def run(self, **kw):
        P.paged_attention(self.q, self.k, self.v, self.table, self.len_t, self.out, window=self.window, sinks=self.sinks,
                          lse=self.lse, **kw)
        torch.cuda.synchronize()
        return self

    def check(self, scale=None, drop=()):
        """Scores are sums of `dim` exact products in fp32, each addition off by 2^-24 of the sum of magnitudes at most, and the
        scaled exponent by 3 further roundings; a weight is off by that, by 2 ulp of ex2.approx (2^-22) and, once a tile, by
        the rescaling's; sums of n weights in fp32 add n 2^-24 at worst, but for 16 keys a tile at a time (n / 16 + 8); the
        weights' second 16 bits leave 2^-16.  Numerator and denominator: twice.  Then the output's own rounding."""
        batch, heads, dim = self.q.shape
        group, half = heads // self.kv, HALF[self.q.dtype]
        scale = dim ** -0.5 if scale is None else scale
        for b, n in enumerate(self.lens):
            keys = [j for j in _visible(n, self.window, self.sinks) if (b, j // self.page) not in drop]
            if not keys:
                assert torch.equal(self.out[b], torch.zeros_like(self.out[b]))
                assert bool((self.lse[b] == -math.inf).all())
                continue
            j = torch.tensor(keys, device=self.q.device)
            at = self.table[b].long()[j // self.page], j % self.page
            k, v = self.k[at].double().repeat_interleave(group, 1), self.v[at].double().repeat_interleave(group, 1)
            q = self.q[b].double()
            s = torch.einsum("hd,nhd->hn", q, k) * scale
            ref = torch.einsum("hn,nhd->hd", torch.softmax(s, 1), v)
            sizes = torch.einsum("hd,nhd->hn", q.abs(), k.abs()).amax(1) * scale
            s_err = (dim + 4) * 2.0 ** -24 * sizes
            w_err = s_err + (len(keys) / 16 + 8) * 2.0 ** -22
            tol = half * ref.abs() + (2 * (w_err + 2.0 ** -16) * v.abs().amax(0).amax(1))[:, None] + 2.0 ** -25
            err = (self.out[b].double() - ref).abs()
            assert bool((err <= tol).all()), f"sequence {b} of {n}: {(err / tol).max().item()} of the tolerance"
            want = torch.logsumexp(s, 1)
            assert bool(((self.lse[b].double() - want).abs() <= w_err + 2.0 ** -22 * (1 + want.abs())).all()), f"lse of {b}"
        assert bool(torch.isnan(self.whole[:, heads:].float()).all() and torch.isnan(self.whole[:, :, dim:].float()).all())


# ---- attention ----------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (8, 2), (16, 1), (40, 2)])
def test_attention_heads_and_types(heads, kv, dim, dtype):
    """One, some, 16 and more than 16 query heads to a key head; both ways to share out the keys."""
    case = Case([1, 0, 130, 17], heads, kv, dim, 16, dtype)
    case.run().check()
    case = Case([1, 0, 130, 17], heads, kv, dim, 16, dtype, wide=4096)      # a wide table: tiles in a row over all CTAs
    case.run().check()


@gpu
@pytest.mark.parametrize("wide", [None, 5000])
@pytest.mark.parametrize("page,order", [(1, "page_slot"), (8, "page_head"), (16, "page_slot"), (64, "page_head"), (256, "page_slot")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 1), (100, 37), (1000, 4)])
def test_attention_pages_and_windows(page, order, window, sinks, wide):
    lens = [63, 64, 65, 1, 127, 200, 0, 500]
    Case(lens, 4, 2, 128, page, torch.bfloat16, window, sinks, order, wide).run().check()


@gpu
@pytest.mark.parametrize("batch,longest", [(1, 5000), (2, 2500), (37, 700), (150, 300)])
def test_attention_long_and_many(batch, longest):
    """Sequences over many CTAs and many sequences to a CTA, of lengths that differ a lot; the same bits each time, and the same
    in every form up to what a form's order of sums allows."""
    rng = random.Random(batch)
    lens = [rng.randint(0, longest) for _ in range(batch - 1)] + [longest]
    case = Case(lens, 8, 2, 64, 16, torch.bfloat16, wide=10000)
    case.run().check()
    first, lse = case.out.clone(), case.lse.clone()
    case.run()
    assert torch.equal(first, case.out) and torch.equal(lse, case.lse)
    case.run(longest=512).check()


@gpu
@pytest.mark.parametrize("longest", [1, 70, 200, 600, None])
def test_attention_cluster_sizes(longest):
    """The hint of the longest length chooses how many CTAs share a sequence; longer ones stay right."""
    Case([1000, 3, 0], 4, 1, 128, 32, torch.float16).run(longest=longest).check()


@gpu
def test_attention_scale_and_large_scores():
    """Scores far apart, so that the running maximum moves, and a scale of the caller's."""
    case = Case([700, 90], 4, 2, 128, 16, torch.bfloat16)
    case.k.mul_(4.0)
    case.run(scale=0.25).check(scale=0.25)


@gpu
@pytest.mark.parametrize("wide", [None, 5000])
def test_attention_keeps_nan_and_infinity_of_a_key(wide):
    """A NaN in a key that is seen reaches the outputs of the heads that read it; a key whose scores are minus infinity weighs
    nothing, and a sequence of such keys alone counts as empty."""
    case = Case([300, 300, 300, 5], 4, 2, 64, 16, torch.bfloat16, wide=wide)
    p0 = case.table[0, 9].item()
    case.k[p0, 3, 1] = float("nan")                                  # sequence 0, key 147, key head 1
    p1 = case.table[1, 2].item()
    case.q[1, :2] = case.q[1, :2].abs() + 0.1
    case.k[p1, 5, 0] = float("-inf")                                 # sequence 1, key 37, key head 0
    case.q[3] = case.q[3].abs() + 0.1
    case.k[case.table[3, 0].item(), :5] = float("-inf")
    case.run()
    nan = torch.isnan(case.out.float()).all(2)
    assert torch.equal(nan, torch.isnan(case.out.float()).any(2))
    assert nan.tolist() == [[False, False, True, True], [False] * 4, [False] * 4, [False] * 4]
    assert torch.isnan(case.lse).tolist() == nan.tolist()
    assert bool((case.out[3] == 0).all()) and bool((case.lse[3] == -math.inf).all())
    keys = torch.tensor([j for j in range(300) if j != 37], device="cuda")
    at = case.table[1].long()[keys // 16], keys % 16
    s = case.k[at][:, 0].double() @ case.q[1, 0].double() / 8
    ref = torch.softmax(s, 0) @ case.v[at][:, 0].double()
    # as in Case.check, with room for positive queries
    assert bool(((case.out[1, 0].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -13 * 8).all())


@gpu
@pytest.mark.parametrize("wide", [None, 5000])
def test_attention_leaves_out_and_reports_bad_pages(wide):
    case = Case([100, 64, 40], 4, 2, 128, 16, torch.bfloat16, wide=wide)
    status = torch.zeros(16, dtype=torch.int32, device="cuda")
    case.run(status=status).check()
    assert status.tolist() == [0] * 16
    case.table[0, 2] = -1
    case.table[1, 1] = case.k.shape[0]
    case.run(status=status).check(drop={(0, 2), (1, 1)})
    assert status[0] == 2 and status[1] == 95 and status[2].item() in (0, 1)
    case.table[2, :3] = -7
    case.run().check(drop={(0, 2), (1, 1), (2, 0), (2, 1), (2, 2)})


@gpu
@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 64])
@pytest.mark.parametrize("wide", [None, 5000])
def test_attention_reports_the_key_of_a_bad_page(page, wide):
    """The record names the sequence and a key of the page, whatever the pages' size."""
    case = Case([5, 16 * 23 + 1], 4, 2, 128, page, torch.bfloat16, wide=wide)
    status = torch.zeros(16, dtype=torch.int32, device="cuda")
    case.table[1, 16 * 23 // page] = -3                                     # that of the last key
    case.run(status=status)
    first = 16 * 23 // page * page
    assert status[:3].tolist() == [2, 95, 1] and first <= status[3].item() <= 16 * 23 and status[4].item() == -3


@gpu
def test_attention_lengths_outside_the_table_are_cut():
    case = Case([64, 64], 2, 1, 64, 16, torch.bfloat16)
    case.run()
    want = case.out.clone()
    case.len_t.copy_(torch.tensor([1000000, 64]))
    case.run()
    assert torch.equal(case.out, want)
    case.len_t.copy_(torch.tensor([-5, 64]))
    case.run()
    assert bool((case.out[0] == 0).all()) and torch.equal(case.out[1], want[1])


@gpu
@pytest.mark.parametrize("page", [4, 8, 16, 64])
@pytest.mark.parametrize("which", ["values first", "one tensor"])
def test_attention_places_of_the_caches(which, page):
    """The values' cache in front of the keys' in memory, and one tensor for both."""
    case = Case([100, 33], 4, 2, 128, page, torch.bfloat16)
    if which == "values first":
        case.k, case.v = case.v, case.k
    else:
        case.v = case.k
    case.run().check()


@gpu
def test_attention_offsets_beyond_32_bits():
    """A cache of more than 4 GiB whose last pages are used (strides that pass 2^31 elements)."""
    pages, page, kv, dim = 70000, 64, 4, 128                         # 2.3e9 elements each: keys and values alias, 4.6 GB
    cache = torch.zeros((pages, page, kv, dim), dtype=torch.bfloat16, device="cuda")
    q = torch.randn((1, kv, dim), device="cuda").to(torch.bfloat16)
    cache[pages - 1] = torch.randn((page, kv, dim), device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([page], dtype=torch.int32, device="cuda")
    P.paged_attention(q, cache, cache, table, lens, out)
    k = cache[pages - 1].double()
    ref = torch.einsum("hn,nhd->hd", torch.softmax(torch.einsum("hd,nhd->hn", q[0].double(), k) * dim ** -0.5, 1), k)
    assert bool(((out[0].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -13 * k.abs().max()).all())


@gpu
def test_attention_on_another_stream_and_in_two_graphs():
    """Calls on a side stream by handle, two calls at once, and two captured graphs replayed on two streams: the workspace of the
    form that needs one is each call's own."""
    cases = [Case([3000, 10, 800], 8, 2, 128, 16, torch.bfloat16, wide=4000, seed=s) for s in range(2)]
    wants = []
    for c in cases:
        c.run().check()
        wants.append(c.out.clone())
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, st in zip(cases, streams):
            P.paged_attention(c.q, c.k, c.v, c.table, c.len_t, c.out, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(c.out, w) for c, w in zip(cases, wants))
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            P.paged_attention(c.q, c.k, c.v, c.table, c.len_t, c.out)
        graphs.append(g)
        c.out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(c.out, w) for c, w in zip(cases, wants))


@gpu
def test_attention_over_its_queries():
    """The output may take the queries' place, in both forms."""
    for wide in (None, 4000):
        case = Case([3000, 10, 0, 800], 8, 2, 128, 16, torch.bfloat16, wide=wide)
        case.run()
        P.paged_attention(case.q, case.k, case.v, case.table, case.len_t, case.q)
        assert torch.equal(case.q, case.out)


@gpu
def test_attention_workspace_on_another_stream_is_its_own():
    """Memory that the current stream still works on is not what a call on another stream gets for its workspace: calls on a side
    stream, between long-running kernels of the current one whose memory has been let go of, give the right answer."""
    case = Case([3000, 10, 800], 8, 2, 128, 16, torch.bfloat16, wide=4000)
    case.run().check()
    want, side = case.out.clone(), torch.cuda.Stream()
    for _ in range(10):
        for n in (1, 2, 4):
            t = torch.full((n << 20,), 7.0, device="cuda")
            for _ in range(20):
                t.mul_(1.0001)
            del t
        P.paged_attention(case.q, case.k, case.v, case.table, case.len_t, case.out, stream=side.cuda_stream)
        side.synchronize()
        assert torch.equal(case.out, want)
        case.out.zero_()
        torch.cuda.synchronize()


@gpu
def test_attention_empty_batch():
    c = Case([5], 2, 1, 64, 16, torch.bfloat16)
    out = c.out[:0]
    assert P.paged_attention(c.q[:0], c.k, c.v, c.table[:0], c.len_t[:0], out) is out


def test_attention_refusals():
    c = Case([40, 3], 4, 2, 64, 16, torch.bfloat16, device="cpu")

    def call(**kw):
        a = dict(q=c.q, k_cache=c.k, v_cache=c.v, block_table=c.table, lens=c.len_t, out=c.out)
        P.paged_attention(**{**a, **kw})
    with pytest.raises(TypeError):
        call(q=c.q.float(), out=c.out.float())
    with pytest.raises(TypeError):
        call(k_cache=c.k.half(), v_cache=c.v.half())
    with pytest.raises(ValueError):
        call(q=c.q[:, :3], out=c.out[:, :3])                    # 3 query heads on 2 key heads
    with pytest.raises(ValueError):
        call(q=c.q[:, :, :32], out=c.out[:, :, :32])
    with pytest.raises(ValueError):
        call(v_cache=c.v.transpose(1, 2).contiguous().transpose(1, 2))   # other strides than the keys
    with pytest.raises(ValueError):
        call(block_table=c.table.long())
    with pytest.raises(ValueError):
        call(block_table=c.table[:1])
    with pytest.raises(ValueError):
        call(lens=c.len_t.long())
    with pytest.raises(ValueError):
        call(lse=torch.zeros(2, 3))
    with pytest.raises(ValueError):
        call(window=-1)
    with pytest.raises(ValueError):
        call(out=c.out[:1].expand(2, -1, -1))
    with pytest.raises(ValueError, match="CUDA device"):
        call()


def test_attention_refuses_a_status_that_is_no_block():
    """A record has 32 bytes; what is smaller, strided or misaligned would be written past."""
    c = Case([40, 3], 4, 2, 64, 16, torch.bfloat16, device="cpu")
    memory = torch.zeros(17, dtype=torch.int32)
    for bad in (memory[:1], memory[:7], memory[1:], memory[::2][:8]):
        with pytest.raises(ValueError, match="status"):
            P.paged_attention(c.q, c.k, c.v, c.table, c.len_t, c.out, status=bad)
    with pytest.raises(ValueError, match="CUDA device"):
        P.paged_attention(c.q, c.k, c.v, c.table, c.len_t, c.out, status=memory[:8])


@gpu
def test_attention_refusals_of_the_native_entry():
    c = Case([40, 3], 4, 2, 64, 16, torch.bfloat16)
    with pytest.raises(RuntimeError, match="power of two"):
        P.paged_attention(c.q, c.k[:, :12], c.v[:, :12], c.table, c.len_t, c.out)
    with pytest.raises(RuntimeError, match="16 bytes"):
        odd = torch.empty((2, 4, 65), dtype=torch.bfloat16, device="cuda")[:, :, 1:]
        P.paged_attention(odd, c.k, c.v, c.table, c.len_t, c.out)
    with pytest.raises(RuntimeError, match="scale"):
        P.paged_attention(c.q, c.k, c.v, c.table, c.len_t, c.out, scale=0.0)
    with pytest.raises(ValueError, match="one device"):
        P.paged_attention(c.q, c.k, c.v, c.table.cpu(), c.len_t, c.out)


def _native_refusal(q, k, v, table, lens, out):
    """What the native entry says to a call that it refuses before it looks for a device (no device needed)."""
    (batch, heads, dim), (pages, size, kv, _) = q.shape, k.shape
    rc = _native.entry("iris_k_paged_attention")(P._ATTENTION.pack(
        *(t.data_ptr() for t in (q, k, v, table, lens, out)), 0, 0, 0, 0, *q.stride()[:2], *k.stride()[:3], table.stride(0),
        *out.stride()[:2], 0, batch, heads, dim, pages, size, kv, table.shape[1], 0, 0, 0, 0, -1, 0, -1, 0, dim ** -0.5))
    lib = _native.kernels()
    lib.iris_paged_attention_last_error.restype = ctypes.c_char_p
    assert rc < 0
    return lib.iris_paged_attention_last_error().decode()


def test_attention_output_that_shares_memory_is_refused():
    """Over a part of the queries, or over the cache; the queries' own place and places beside them are none of that."""
    c = Case([40, 3], 4, 2, 64, 16, torch.bfloat16, device="cpu")
    rows = torch.zeros((4, 8, 2, 64), dtype=torch.bfloat16)
    q, fine = rows[:2, :4, 0], "no device"
    a = (q, c.k, c.v, c.table, c.len_t)
    assert fine in _native_refusal(*a, q)
    assert fine in _native_refusal(*a, rows[:2, :4, 1])      # between the heads
    assert fine in _native_refusal(*a, rows[:2, 4:, 0])      # beside them
    assert fine in _native_refusal(*a, rows[2:, :4, 0])
    for bad in (rows[1:3, :4, 0], rows[:2, 1:5, 0], rows.flatten(1)[:2, 32:544].unflatten(1, (4, 128))[:, :, :64],
                rows[:2].flatten(1)[:, :256].unflatten(1, (4, 64))):
        assert "share no memory" in _native_refusal(*a, bad)
    flat = torch.as_strided(c.k, (c.k.numel(),), (1,), c.k.storage_offset())
    assert "cache" in _native_refusal(*a, flat[:512].view(2, 4, 64))


def test_attention_outputs_that_share_memory_with_anything_are_refused():
    """Heads of the output that meet one another, and sums or outputs over any other array; places between and beside are fine.
    (By the native entry, before it looks for a device.)"""
    c = Case([40, 3, 8], 4, 2, 64, 16, torch.bfloat16, device="cpu")
    flat = torch.zeros(4096, dtype=torch.bfloat16)

    def answer(q=c.q, out=c.out, lse=None, table=c.table, lens=c.len_t):
        (batch, heads, dim), (pages, size, kv, _) = q.shape, c.k.shape
        lse_at, lse_pitch = (0, 0) if lse is None else (lse.data_ptr(), lse.stride(0))
        rc = _native.entry("iris_k_paged_attention")(P._ATTENTION.pack(
            *(t.data_ptr() for t in (q, c.k, c.v, table, lens, out)), lse_at, 0, 0, 0, *q.stride()[:2], *c.k.stride()[:3],
            table.stride(0), *out.stride()[:2], lse_pitch, batch, heads, dim, pages, size, kv, table.shape[1], 0, 0, 0, 0, -1, 0,
            -1, 0, dim ** -0.5))
        lib = _native.kernels()
        lib.iris_paged_attention_last_error.restype = ctypes.c_char_p
        assert rc < 0
        return lib.iris_paged_attention_last_error().decode()
    heads = lambda *pitches: torch.as_strided(flat, (3, 4, 64), (*pitches, 1), 0)   # noqa: E731
    for fine in (heads(256, 64), heads(64, 192), heads(128, 512), heads(1024, 72)):
        assert "no device" in answer(out=fine)
    for bad in (heads(64, 64), heads(64, 128), heads(128, 64), heads(192, 64), heads(256, 80)):
        assert "must not overlap" in answer(out=bad)
    wide = torch.zeros((3, 8), dtype=torch.float32)
    assert "no device" in answer(lse=wide[:, :4])
    assert "must not overlap" in answer(lse=wide[:1, :4].expand(3, -1))
    floats = lambda t: torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0).view(torch.float32)   # noqa: E731
    for other in (c.q, c.k, c.out):
        at = floats(other)[other.storage_offset() // 2:][:12].view(3, 4)
        assert "lse must share" in answer(lse=at), other.shape
    at = floats(c.whole)[128:224].view(3, 32)[:, :4]                              # within what the views' first and last bytes span
    assert "lse must share" in answer(lse=at)
    gap = torch.as_strided(floats(c.whole), (3, 4), (5 * 36, 1), 4 * 36)           # behind the last head of a sequence
    assert "no device" in answer(out=c.out[:, :, :], lse=gap.clone())


@gpu
def test_attention_outputs_over_the_table_or_the_lengths_are_refused():
    c = Case([40, 3, 8], 4, 2, 64, 16, torch.bfloat16)
    flat, wide = torch.zeros(4096, dtype=torch.bfloat16, device="cuda"), torch.zeros((3, 8), device="cuda")
    ints, out = flat.view(torch.int32), flat[:768].view(3, 4, 64)
    ok = dict(q=c.q, k_cache=c.k, v_cache=c.v, block_table=c.table, lens=c.len_t, out=c.out)
    for bad in (dict(lse=torch.as_strided(c.table, (12,), (1,), 0).view(torch.float32).view(3, 4)),
                dict(lse=wide[:, :4], lens=wide.view(torch.int32).flatten()[1:4]),
                dict(out=out, block_table=ints[40:58].view(3, 6)), dict(out=out, lens=ints[:3])):
        with pytest.raises(RuntimeError, match="block table or the lengths"):
            P.paged_attention(**{**ok, **bad})
    P.paged_attention(**{**ok, "lse": wide[:, :4], "lens": wide.view(torch.int32).flatten()[4:7]})   # between the rows: lengths of zero
    assert not c.out.any() and bool((wide[:, :4] == -math.inf).all()) and not wide[:, 4:].any()


def test_attention_table_of_too_many_keys_is_refused():
    """Positions are counted in 32 bits, up to a batch of blocks behind the last key."""
    c = Case([40, 3], 4, 2, 64, 16, torch.bfloat16, device="cpu")
    wide = 2 ** 27
    table = torch.as_strided(torch.zeros(1, dtype=torch.int32), (2, wide), (0, 0))
    assert "2^31" in _native_refusal(c.q, c.k, c.v, table, c.len_t, c.out)
    assert "no device" in _native_refusal(c.q, c.k, c.v, table[:, :wide - 64], c.len_t, c.out)


@gpu
def test_attention_whose_waits_may_run_out():
    """A limit of a microsecond: the call comes back, with or without having recorded that a wait ran out, with no copy left on its
    way, and the next one is right."""
    for wide, batch in ((None, 5), (8000, 5), (8000, 300)):
        case = Case([3000, 10, 800, 0, 77] * (batch // 5), 8, 2, 128, 16, torch.bfloat16, wide=wide)
        status = torch.zeros(64, dtype=torch.int32, device="cuda")
        for _ in range(20):
            P.paged_attention(case.q, case.k, case.v, case.table, case.len_t, case.out, timeout_ms=1e-3, status=status)
        torch.cuda.synchronize()
        assert status[0].item() in (0, 1), status[:8]
        case.run().check()


@gpu
@pytest.mark.parametrize("wide", [None, 5000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_weights_far_below_the_largest_count(dtype, wide):
    """One key takes nearly all of the weight and has values of zero; 20000 others of weight exp(-18) = 2^-25.97 each make up the
    output.  Scores are one exact product, the exponent 26 is off by a few 2^-24 of itself and a weight by ex2's 2^-22 besides, sums
    of n equal weights in fp32 by (n / 16 + 8) 2^-22 at worst, the weights' second 16 bits leave 2^-16; the output is rounded once."""
    n, dominant = 20000, 77
    case = Case([n, 3], 4, 2, 64, 16, dtype, wide=wide)
    case.q[0].zero_()
    case.q[0, :, 0] = 8.0
    j = torch.arange(n, device="cuda")
    at = case.table[0].long()[j // 16], j % 16
    case.k[at] = 0.0
    case.v[at] = 1.0
    page = case.table[0, dominant // 16].item()
    case.k[page, dominant % 16, :, 0] = 18.0
    case.v[page, dominant % 16] = 0.0
    case.run()
    others = (n - 1) * math.exp(-18.0)
    want, rel = others / (1 + others), HALF[dtype] + (n / 16 + 8) * 2.0 ** -22 + 2.0 ** -16 + 2.0 ** -17
    assert bool(((case.out[0].double() - want).abs() <= rel * want).all()), (case.out[0, 0, 0].item(), want)
    assert bool(((case.lse[0].double() - (18.0 + math.log1p(others))).abs() <= 2.0 ** -22 * 20 + rel * others).all())


@gpu
@pytest.mark.parametrize("wide", [None, 5000])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_huge_scores_stays_finite(sign, wide):
    """fp16, scores of up to 2^27 (in powers of two) of either sign, each off by as much as 4: one key of each sequence is
    far above the others, so that its values are the output (to a weight's 2^-16 and the output's rounding)."""
    lens = [200 + 37 * i for i in range(12)]
    case = Case(lens, 4, 2, 64, 16, torch.float16, wide=wide, seed=5)
    g = torch.Generator().manual_seed(11)
    want = torch.empty((12, 4, 64), dtype=torch.float64, device="cuda")
    case.q.zero_()
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        at = case.table[b].long()[j // 16], j % 16
        size = float(torch.randint(4000, 30000, (1,), generator=g))
        case.q[b, :, 0] = 2000.0 + 97 * b
        case.k[at] = 0.0
        case.k[at[0], at[1], :, 0] = size / 2 if sign > 0 else -2 * size
        top = int(torch.randint(0, n, (1,), generator=g))
        case.k[at[0][top], at[1][top], :, 0] = size * sign
        want[b] = case.v[at[0][top], at[1][top]].double().repeat_interleave(2, 0)
    case.run(scale=1.0)
    assert bool(((case.out.double() - want).abs() <= (HALF[torch.float16] + 2.0 ** -15) * want.abs()).all())


# ---- pages --------------------------------------------------------------------------------------------------------------

def _plain_reserve(lens, new, table, free, count, page, rows, row_stride):
    """The requests one after the other, as the documentation says it."""
    wide = len(table[0])
    slots, positions = [-1] * rows, [-1] * rows
    lens, table, left, start, out_of_pages = list(lens), [list(r) for r in table], count, 0, False
    sums = 0
    for b, (n, more) in enumerate(zip(list(lens), new)):
        n, more = max(n, 0), max(more, 0)
        row = b * row_stride if row_stride else start
        start += more
        fits = n + more <= wide * page and (more <= row_stride if row_stride else start <= rows)
        if not fits:
            continue
        held = -(-n // page)
        need = -(-(n + more) // page) - held
        sums += need
        if need and sums > count:
            continue
        for i in range(need):
            left -= 1
            table[b][held + i] = free[left]
        lens[b] = n + more
        for j in range(more):
            pos = n + j
            slots[row + j], positions[row + j] = table[b][pos // page] * page + pos % page, pos
    return slots, positions, table, lens, left


def _state(batch, page, wide, most, seed, short=None):
    rng = random.Random(seed)
    lens = [rng.choice((0, 1, page, rng.randint(0, wide * page))) for _ in range(batch)]
    new = [rng.choice((0, 1, most, rng.randint(0, most))) for _ in range(batch)]
    held = [min(wide, -(-n // page)) for n in lens]
    ids = list(range(sum(held) + batch * wide))
    rng.shuffle(ids)
    table = [[ids.pop() if i < h else -1 for i in range(wide)] for h in held]
    count = len(ids) if short is None else min(len(ids), short)
    return lens, new, table, ids, count


@gpu
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("batch,page,wide,most,short", [
    (1, 16, 1, 1, None), (1, 1, 40, 7, None), (5, 16, 8, 40, None), (5, 16, 8, 40, 3), (512, 16, 10, 1, None),
    (513, 16, 10, 3, 100), (700, 4, 9, 20, 40), (1300, 64, 4, 130, None), (1300, 64, 4, 130, 0), (3, 128, 50, 3000, None)])
def test_reserve(batch, page, wide, most, short, packed, in_place):
    lens, new, table, free, count = _state(batch, page, wide, most, batch + most, short)
    rows = sum(new) + 5 if packed else batch * most + 3
    stride = 0 if packed else most
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    spare = torch.full((batch, wide + 2), -9, dtype=torch.int32, device="cuda")
    spare[:, 1:-1] = i32(table)
    table_t, lens_t, count_t = spare[:, 1:-1], i32(lens), i32([count])
    slots, positions = i32([-7] * rows), i32([-7] * rows)
    lens_out, count_out = (None, None) if in_place else (i32([0] * batch), i32([0]))
    P.reserve_slots(lens_t, i32(new), table_t, i32(free), count_t, page, slots, positions, row_stride=stride, lens_out=lens_out,
                    free_count_out=count_out)
    want = _plain_reserve(lens, new, table, free, count, page, rows, stride)
    got = (slots, positions, table_t, lens_t if in_place else lens_out, count_t if in_place else count_out)
    for name, g, w in zip(("slots", "positions", "table", "lengths", "count"), got, want):
        assert g.tolist() == ([w] if name == "count" else w), name
    if not in_place:
        assert lens_t.tolist() == lens and count_t.tolist() == [count]
    assert bool((spare[:, 0] == -9).all()) and bool((spare[:, -1] == -9).all())


@gpu
def test_reserve_packed_rows_that_do_not_last():
    """Packed requests behind the last row get nothing, those that fit do."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    lens, table, count = i32([0, 0, 0]), i32([[-1] * 4] * 3), i32([9])
    slots, positions = i32([5] * 10), i32([5] * 10)
    P.reserve_slots(lens, i32([4, 7, 0]), table, i32(list(range(9))), count, 4, slots, positions)
    assert lens.tolist() == [4, 0, 0] and count.tolist() == [8] and slots.tolist() == [32, 33, 34, 35] + [-1] * 6


@gpu
@pytest.mark.parametrize("batch,page,wide", [(1, 16, 3), (40, 16, 8), (1100, 8, 5)])
def test_release_gives_everything_back(batch, page, wide):
    lens, new, table, free, count = _state(batch, page, wide, 1, batch)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    held = [min(wide, -(-n // page)) for n in lens]
    which = [b % 3 != 1 for b in range(batch)]
    free = free[:count]
    free_t = i32(free + [-5] * sum(held))
    lens_t, table_t, count_t = i32(lens), i32(table), i32([count])
    P.release_slots(lens_t, i32([int(w) for w in which]), table_t, free_t, count_t, page)
    back = [table[b][i] for b in range(batch) if which[b] for i in range(held[b])]
    assert count_t.tolist() == [count + len(back)]
    assert free_t.tolist() == free + back + [-5] * (sum(held) - len(back))
    assert lens_t.tolist() == [0 if w else n for n, w in zip(lens, which)]
    assert table_t.tolist() == [[-1] * wide if w else r for r, w in zip(table, which)]
    P.release_slots(lens_t, i32([1] * batch), table_t, free_t, count_t, page)
    assert count_t.tolist() == [count + sum(held)]
    assert sorted(free_t.tolist()) == sorted(free + [i for r in table for i in r if i >= 0])
    assert lens_t.tolist() == [0] * batch


@gpu
@pytest.mark.parametrize("batch", [4, 700])
def test_release_takes_any_number_but_zero_for_yes(batch):
    """``which`` may be the negative of a comparison, or bits."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    which = [(-1, 0, -(2 ** 31), 7)[b % 4] for b in range(batch)]
    lens, table, free, count = i32([3] * batch), i32([[b] for b in range(batch)]), i32([-5] * batch), i32([0])
    P.release_slots(lens, i32(which), table, free, count, 4)
    back = [b for b in range(batch) if which[b]]
    assert lens.tolist() == [0 if w else 3 for w in which] and count.item() == len(back)
    assert free.tolist() == back + [-5] * (batch - len(back))
    assert table.flatten().tolist() == [-1 if w else b for b, w in enumerate(which)]


@gpu
def test_release_without_room_keeps_the_request():
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    lens, table, free, count = i32([8, 8, 8]), i32([[1, 2], [3, 4], [5, 6]]), i32([0, 9, 9, 9]), i32([1])
    P.release_slots(lens, i32([1, 1, 1]), table, free, count, 4)
    assert lens.tolist() == [0, 8, 8] and count.tolist() == [3] and free.tolist() == [0, 1, 2, 9]
    assert table.tolist() == [[-1, -1], [3, 4], [5, 6]]


@gpu
@pytest.mark.parametrize("batch,page,wide,holes", [
    (1, 16, 3, 1), (40, 16, 8, 30), (600, 4, 20, 4000), (1100, 8, 5, 1500), (3, 1, 20000, 9000), (2100, 2, 3, 0)])
def test_release_passes_over_entries_that_are_no_page(batch, page, wide, holes):
    """Pages that a program took out of a request's row itself (negative entries) are not put on the list of free pages; the others
    go back in their order, and room is needed for them alone."""
    lens, new, table, free, count = _state(batch, page, wide, 1, batch)
    rng = random.Random(holes)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    held = [min(wide, -(-n // page)) for n in lens]
    for _ in range(holes):
        b = rng.randrange(batch)
        if held[b]:
            table[b][rng.randrange(held[b])] = rng.choice((-1, -7, -(2 ** 31)))
    which = [b % 3 != 1 for b in range(batch)]
    free = free[:count]
    back = [table[b][i] for b in range(batch) if which[b] for i in range(held[b]) if table[b][i] >= 0]
    free_t, lens_t, table_t, count_t = i32(free + [-5] * len(back)), i32(lens), i32(table), i32([count])
    P.release_slots(lens_t, i32([int(w) for w in which]), table_t, free_t, count_t, page)
    assert count_t.tolist() == [count + len(back)]
    assert free_t.tolist() == free + back
    assert lens_t.tolist() == [0 if w else n for n, w in zip(lens, which)]
    assert table_t.tolist() == [[-1] * wide if w else r for r, w in zip(table, which)]


@gpu
def test_release_without_room_counts_pages_alone():
    """A row without pages needs no room, also behind a request that finds none."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    lens, table, free, count = i32([8, 8, 8, 8]), i32([[1, -1], [-1, 4], [5, 6], [-3, -3]]), i32([0, 9, 9, 9]), i32([1])
    P.release_slots(lens, i32([1, 1, 1, 1]), table, free, count, 4)
    assert lens.tolist() == [0, 0, 8, 0] and count.tolist() == [3] and free.tolist() == [0, 1, 4, 9]
    assert table.tolist() == [[-1, -1], [-1, -1], [5, 6], [-1, -1]]


@gpu
def test_cache_lives_through_requests():
    """Requests that come, grow and go for many steps: no page is ever held twice, and none is lost."""
    rng = random.Random(3)
    cache = P.PagedCache(1, 50, 16, 1, 64, 6, 200, device="cuda")
    slots, positions = (torch.empty(6 * 40, dtype=torch.int32, device="cuda") for _ in range(2))
    refused = 0
    for step in range(60):
        new = torch.tensor([rng.choice((0, 1, 40)) for _ in range(6)], dtype=torch.int32, device="cuda")
        before = cache.lens.clone()
        cache.reserve(new, slots, positions, row_stride=40)
        refused += int(((cache.lens == before) & (new > 0)).sum())
        if rng.random() < 0.3:
            cache.release(torch.tensor([int(rng.random() < 0.4) for _ in range(6)], dtype=torch.int32, device="cuda"))
        held = [p for b, n in enumerate(cache.lens.tolist()) for p in cache.block_table[b, :-(-n // 16)].tolist()]
        free = cache.free_pages[:int(cache.free_count)].tolist()
        assert sorted(held + free) == list(range(50)), step
    assert refused > 0


@pytest.mark.parametrize("name,bad", [
    ("slots", "positions"), ("positions", "lens"), ("slots", "free_pages"), ("lens_out", "free_pages"), ("slots", "block_table"),
    ("count_out", "new_lens"), ("lens", "block_table")])
def test_reserve_whose_arrays_share_memory_is_refused(name, bad):
    """By the native entry, before it looks for a device (none needed)."""
    memory = torch.zeros(400, dtype=torch.int32)
    sizes = dict(lens=3, new_lens=3, block_table=24, free_pages=9, free_count=1, slots=12, positions=12, lens_out=3, count_out=1)
    at = {n: memory.data_ptr() + 160 * i for i, n in enumerate(sizes)}
    at[name] = at[bad] + 4 * max(0, sizes[bad] - 1 - 4 * (bad == "block_table"))
    rc = _native.entry("iris_k_reserve_slots")(P._RESERVE.pack(
        *(at[n] for n in ("lens", "new_lens", "block_table", "free_pages", "free_count", "slots", "positions", "lens_out", "count_out")),
        0, 8, 4, 9, 16, 3, 12, 0))
    lib = _native.kernels()
    lib.iris_pages_last_error.restype = ctypes.c_char_p
    assert rc == -1 and "share memory" in lib.iris_pages_last_error().decode()


@pytest.mark.parametrize("name,other,fine", [
    ("free_pages", "block_table", False), ("free_pages", "lens", False), ("free_pages", "which", False), ("free_count", "free_pages", False),
    ("lens", "block_table", False), ("which", "block_table", False), ("free_count", "lens", False), ("free_count", "gap", True),
    ("which", "gap", True), ("lens", "gap", True), ("which", "whole lens", True), ("lens", "part of which", False)])
@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused must find no device")
def test_release_whose_arrays_share_memory_is_refused(name, other, fine):
    """By the native entry, before it looks for a device; places in the gaps of a strided table, and the lengths as `which`, are fine."""
    memory = torch.zeros(400, dtype=torch.int32)
    sizes = dict(lens=3, which=3, block_table=24, free_pages=9, free_count=1)
    at = {n: memory.data_ptr() + 160 * i for i, n in enumerate(sizes)}
    if other == "gap":
        at[name] = at["block_table"] + 4 * 12                       # rows of 4 at 8 to 11 and 16 to 19
    elif other == "whole lens":
        at[name] = at["lens"]
    elif other == "part of which":
        at[name] = at["which"] + 8
    else:
        at[name] = at[other] + 4 * (max(0, sizes[other] - 1 - 4 * (other == "block_table")))
    lib = _native.kernels()
    rc = _native.typed(lib.iris_k_release_slots, P._RELEASE)(
        at["lens"], at["which"], at["block_table"], 8, 4, at["free_pages"], 9, at["free_count"], 16, 3, 0)
    lib.iris_pages_last_error.restype = ctypes.c_char_p
    assert ("share memory" in lib.iris_pages_last_error().decode()) == (not fine) and rc == (-3 if fine else -1)


@gpu
def test_reserve_lengths_over_the_new_ones_and_arrays_between_the_rows():
    """``lens_out`` may be ``new_lens``, and a count or lengths may lie in the gaps of a strided table; ``which`` may be the lengths."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    for batch in (3, 700, 2500):
        whole = torch.full((batch, 9), -1, dtype=torch.int32, device="cuda")
        table, count, free = whole[:, :4], whole[1, 5:6], i32(list(range(2 * batch)))
        count.fill_(2 * batch)
        lens, new, rows = i32([0] * batch), i32([1 + b % 2 * 4 for b in range(batch)]), sum(1 + b % 2 * 4 for b in range(batch))
        slots, positions = i32([0] * rows), i32([0] * rows)
        P.reserve_slots(lens, new, table, free, count, 4, slots, positions, lens_out=new)
        assert new.tolist() == [1 + b % 2 * 4 for b in range(batch)] and not lens.any()
        taken = sum(1 + b % 2 for b in range(batch))
        assert count.item() == 2 * batch - taken
        pages = []
        for b in range(batch):   # one page, two pages, one page, ..
            first = 3 * (b // 2) + b % 2
            pages.append([2 * batch - 1 - i for i in range(first, first + 1 + b % 2)])
        assert [r[:len(p)] for r, p in zip(table.tolist(), pages)] == pages
        P.release_slots(new, new, table, free, count, 4)
        assert count.item() == 2 * batch and not new.any() and bool((table == -1).all())
        assert sorted(free.tolist()) == list(range(2 * batch))


@gpu
@pytest.mark.parametrize("row_stride", [0, 40])
def test_reserve_stops_at_the_longest_length(row_stride):
    """``max_len`` binds although the last page has room for more, and a request beyond it is in nobody's way."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    cache = P.PagedCache(1, 20, 16, 1, 64, 3, 35, device="cuda")
    slots, positions = i32([0] * 120), i32([0] * 120)
    cache.reserve(i32([35, 34, 36]), slots, positions, row_stride=row_stride)
    assert cache.lens.tolist() == [35, 34, 0] and cache.free_count.item() == 14
    cache.reserve(i32([1, 1, 35]), slots, positions, row_stride=row_stride)
    assert cache.lens.tolist() == [35, 35, 35] and cache.free_count.item() == 11
    first = row_stride or 1
    assert positions[0].item() == -1 and slots[0].item() == -1 and positions[first].item() == 34
    cache.reserve(i32([1, 0, 2]), slots, positions, row_stride=row_stride)
    assert cache.lens.tolist() == [35, 35, 35] and bool((positions == -1).all())
    table, lens, count = i32([[-1] * 4]), i32([0]), i32([9])
    for limit, want in ((3, 0), (4, 4), (None, 8)):
        P.reserve_slots(lens, i32([4]), table, i32(list(range(9))), count, 4, slots, positions, max_len=limit)
        assert lens.item() == want


def test_reserve_refuses_a_negative_longest_length():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)   # noqa: E731
    with pytest.raises(ValueError, match="max_len"):
        P.reserve_slots(i32(3), i32(3), i32(3, 4), i32(9), i32(1), 16, i32(12), i32(12), max_len=-1)


@gpu
@pytest.mark.parametrize("batch", [4, 700])
def test_reserve_for_requests_that_hold_nothing(batch):
    """``fresh``: a request that holds tokens gets nothing, takes no page, and is in nobody's way."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    held = [b % 2 * 5 for b in range(batch)]
    table = [[b, -1] if held[b] else [-1, -1] for b in range(batch)]
    lens, table_t, count = i32(held), i32(table), i32([batch])
    slots, positions = i32([7] * 6 * batch), i32([7] * 6 * batch)
    new = [6 - b % 4 // 2 * 6 for b in range(batch)]            # 6, 6, 0, 0, ..
    P.reserve_slots(lens, i32(new), table_t, i32(list(range(batch, 2 * batch))), count, 8, slots, positions, row_stride=6, fresh=True)
    given = [b for b in range(batch) if new[b] and not held[b]]
    assert lens.tolist() == [6 if b in given else held[b] for b in range(batch)]
    assert count.item() == batch - len(given)
    pages = {b: 2 * batch - 1 - i for i, b in enumerate(given)}
    assert table_t.tolist() == [[pages[b], -1] if b in pages else table[b] for b in range(batch)]
    want = [[pages[b] * 8 + j if b in pages else -1 for j in range(6)] for b in range(batch)]
    assert slots.view(batch, 6).tolist() == want
    assert positions.view(batch, 6).tolist() == [list(range(6)) if b in pages else [-1] * 6 for b in range(batch)]


def test_reserve_refusals():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)   # noqa: E731
    ok = dict(lens=i32(3), new_lens=i32(3), block_table=i32(3, 4), free_pages=i32(9), free_count=i32(1), page_size=16,
              slots=i32(12), positions=i32(12))
    for bad in (dict(lens=i32(3).long()), dict(new_lens=i32(2)), dict(block_table=i32(2, 4)), dict(block_table=i32(4, 3).t()),
                dict(free_count=i32(2)), dict(page_size=12), dict(page_size=0), dict(positions=i32(11)), dict(row_stride=5),
                dict(row_stride=-1), dict(lens_out=i32(2)), dict(slots=i32(24)[::2])):
        with pytest.raises(ValueError):
            P.reserve_slots(**{**ok, **bad})
    with pytest.raises(ValueError, match="CUDA device"):
        P.reserve_slots(**ok)
    ok = dict(lens=i32(3), which=i32(3), block_table=i32(3, 4), free_pages=i32(9), free_count=i32(1), page_size=16)
    for bad in (dict(which=i32(3).bool()), dict(block_table=i32(3)), dict(page_size=3)):
        with pytest.raises(ValueError):
            P.release_slots(**{**ok, **bad})
    with pytest.raises(ValueError):
        P.PagedCache(1, 8, 12, 1, 64, 1, 100)
    with pytest.raises(TypeError):
        P.PagedCache(1, 8, 16, 1, 64, 1, 100, dtype=torch.float32)
