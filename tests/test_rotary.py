"""Head norms, rotation and cache writes against the formulas in 64 bits, the table of angles, and the refusals."""
import ctypes
import math

import pytest
import torch

from iris_b200 import _native
from iris_b200.ops import rotary as R

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of a rounding, relative


def _turn(x, pos, table, interleaved):
    """x [tokens, heads, dim] in 64 bits, rotated; and for every component the magnitudes that were added up for it."""
    rot = table.shape[1]
    c, s = (t[:, None] for t in table[pos].double().split(rot // 2, 1))
    first = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    second = first + 1 if interleaved else first + rot // 2
    first, second = first.to(x.device), second.to(x.device)
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return y, size


class Case:
    def __init__(self, tokens, heads, kv, dim, rot, dtype, norm=True, interleaved=False, page=16, order="page_slot", seed=0,
                 device="cuda"):
        g = torch.Generator().manual_seed(seed + tokens + dim)
        self.heads, self.kv, self.dim, self.interleaved, self.page = heads, kv, dim, interleaved, page
        width = (heads + 2 * kv) * dim
        self.qkv = (torch.randn((tokens, width + 24), generator=g) * 3).to(device, dtype)[:, 8:8 + width]
        self.w = [(1 + 0.2 * torch.randn(dim, generator=g)).to(device, dtype) if norm else None for _ in range(2)]
        self.table = R.rotary_table(500, rot).to(device)
        self.pos = torch.randint(0, 500, (tokens,), generator=g).to(device, torch.int32)
        pages = math.ceil(tokens / page) + 2
        data = torch.full((2, pages, kv, page, dim) if order == "page_head" else (2, pages, page, kv, dim), float("nan"))
        data = data.to(device, dtype)
        self.k, self.v = data.transpose(2, 3) if order == "page_head" else data
        self.slots = torch.randperm(pages * page, generator=g)[:tokens].to(device, torch.int32)
        self.whole = torch.full((tokens + 1, width + 16), float("nan"), dtype=dtype, device=device)
        self.out = self.whole[:tokens, 8:8 + width]

    def kw(self):
        return dict(q_weight=self.w[0], k_weight=self.w[1], interleaved=self.interleaved)

    def cache(self):
        return dict(k_cache=self.k, v_cache=self.v, slots=self.slots)

    def want(self, eps=1e-6):
        x = self.qkv.double().unflatten(1, (-1, self.dim))
        parts, sizes = [], []
        for part, w in ((x[:, :self.heads], self.w[0]), (x[:, self.heads:self.heads + self.kv], self.w[1])):
            if w is not None:
                part = part * torch.rsqrt(part.square().mean(2, keepdim=True) + eps) * w.double()
            y, size = _turn(part, self.pos.long().clamp(0, 499), self.table, self.interleaved)
            parts.append(y), sizes.append(size)
        return torch.cat(parts + [x[:, self.heads + self.kv:]], 1), torch.cat(sizes, 1)

    def close(self, got, want, size):
        """fp32: a lane adds 16 squares and the lanes' sums, 22 roundings of 2^-24 at most, half of that in the root; rsqrt and
        the products 2^-22; the rotation four roundings of the magnitudes added; 2^-20 in all.  Then one rounding to 16 bits."""
        tol = HALF[got.dtype] * want.abs() + 2.0 ** -20 * size + 2.0 ** -25
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), (err / tol).max().item()

    def check(self, rows=None, cached=None):
        want, size = self.want()
        tokens = want.shape[0]
        rows = torch.ones(tokens, dtype=torch.bool) if rows is None else rows
        cached = rows if cached is None else cached
        n = self.heads + self.kv
        if self.out is not None:
            got = self.out.unflatten(1, (-1, self.dim))
            self.close(got[rows][:, :min(n, got.shape[1])], want[rows][:, :min(n, got.shape[1])], size[rows][:, :min(n, got.shape[1])])
            if got.shape[1] > n:
                assert torch.equal(got[rows][:, n:].double(), want[rows][:, n:])
        written = torch.zeros(self.k.shape[:2], dtype=torch.bool, device=self.k.device)
        at = self.slots[cached].long()
        written[at // self.page, at % self.page] = True
        self.close(self.k[at // self.page, at % self.page], want[cached][:, self.heads:n], size[cached][:, self.heads:n])
        assert torch.equal(self.v[at // self.page, at % self.page].double(), want[cached][:, n:])
        for t in (self.k, self.v):
            assert bool(torch.isnan(t[~written].float()).all()), "wrote outside the slots"


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", ["page_slot", "page_head"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(16, 16), (64, 64), (80, 32), (96, 96), (128, 128), (128, 48), (256, 64), (512, 512), (272, 16)])
def test_every_head_size(dim, rot, interleaved, order, dtype):
    for heads, kv, norm in ((5, 1, True), (4, 4, False)):
        c = Case(33, heads, kv, dim, rot, dtype, norm, interleaved, order=order)
        R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, heads, kv, dim, **c.kw(), **c.cache())
        c.check()
        assert bool(torch.isnan(c.whole[-1].float()).all() and torch.isnan(c.whole[:, :8].float()).all() and
                    torch.isnan(c.whole[:, 8 + c.out.shape[1]:].float()).all())


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 1000])
@pytest.mark.parametrize("heads,kv", [(1, 1), (64, 8), (200, 3)])
def test_tokens_and_heads(tokens, heads, kv):
    c = Case(tokens, heads, kv, 128, 128, torch.bfloat16)
    R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, heads, kv, 128, **c.kw(), **c.cache())
    c.check()
    # the queries alone: the same bits, and the same cache
    out = torch.empty((tokens, heads * 128), dtype=torch.bfloat16, device="cuda")
    k = c.k.clone()
    c.k.fill_(float("nan")), c.v.fill_(float("nan"))
    R.qk_norm_rope(c.qkv, out, c.pos, c.table, heads, kv, 128, **c.kw(), **c.cache())
    assert torch.equal(out, c.out[:, :heads * 128]) and torch.equal(k.nan_to_num(9.0), c.k.nan_to_num(9.0))
    # in place, without a cache: the same bits, values untouched
    whole = c.out.clone()
    x = c.qkv
    assert R.qk_norm_rope(x, x, c.pos, c.table, heads, kv, 128, **c.kw()) is x
    assert torch.equal(x, whole)


@gpu
def test_one_weight_alone_and_eps():
    c = Case(40, 3, 2, 64, 32, torch.float16)
    c.w[0] = None
    R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 3, 2, 64, **c.kw(), **c.cache())
    c.check()
    c = Case(40, 3, 2, 64, 32, torch.float16)
    c.qkv.zero_()                                             # a head of zeros stays one
    R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 3, 2, 64, **c.kw(), **c.cache())
    assert bool((c.out == 0).all())


@gpu
@pytest.mark.parametrize("dim", [96, 128])
def test_rows_of_no_token_stay_as_they_were(dim):
    c = Case(50, 4, 2, dim, dim, torch.bfloat16)
    c.pos[7] = -1
    c.slots[11] = -1
    c.slots[7] = c.slots[0]                                   # (a row without a position writes nothing)
    status = torch.zeros(16, dtype=torch.int32, device="cuda")
    R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 4, 2, dim, **c.kw(), **c.cache(), status=status)
    rows = torch.ones(50, dtype=torch.bool)
    rows[7] = False
    cached = rows.clone()
    cached[11] = False
    c.check(rows, cached)
    assert bool(torch.isnan(c.out[7].float()).all()) and status.tolist() == [0] * 16


@gpu
@pytest.mark.parametrize("what", ["position", "slot"])
def test_positions_and_slots_out_of_range_are_skipped_and_reported(what):
    c = Case(50, 4, 2, 64, 64, torch.bfloat16)
    rows, cached = torch.ones(50, dtype=torch.bool), torch.ones(50, dtype=torch.bool)
    if what == "position":
        c.pos[20] = 500
        rows[20] = cached[20] = False
    else:
        c.slots[20] = c.k.shape[0] * 16
        cached[20] = False
    status = torch.zeros(16, dtype=torch.int32, device="cuda")
    R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 4, 2, 64, **c.kw(), **c.cache(), status=status)
    c.check(rows, cached)
    assert status[0] == 2 and status[1] == (96 if what == "position" else 97) and status[3] == 20
    if what == "position":
        assert bool(torch.isnan(c.out[20].float()).all())


@gpu
def test_in_a_graph_and_on_another_stream():
    c = Case(60, 4, 2, 128, 128, torch.bfloat16)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 4, 2, 128, **c.kw(), **c.cache(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    c.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 4, 2, 128, **c.kw(), **c.cache())
    c.qkv.mul_(0.5), c.pos.add_(-1).clamp_(min=0)
    g.replay()
    torch.cuda.synchronize()
    c.check()


@gpu
@pytest.mark.parametrize("norm", [True, False])
def test_without_rotation(norm):
    """No table: norms and cache writes alone, positions as large as they come; nothing at all to do leaves every bit."""
    c = Case(70, 4, 2, 128, 128, torch.bfloat16, norm)
    c.table = torch.cat([torch.ones(500, 64), torch.zeros(500, 64)], 1).cuda()      # for the comparison: angles of zero
    pos = c.pos + 2000000000
    R.qk_norm_rope(c.qkv, c.out, pos, None, 4, 2, 128, **c.kw(), **c.cache())
    c.check()
    assert norm or torch.equal(c.out, c.qkv)


@gpu
def test_offsets_beyond_32_bits():
    """A matrix of more than 2^31 elements, in place: its last rows have the bits of the same rows alone."""
    tokens, heads = 180000, 32
    width = 3 * heads * 128
    qkv = torch.zeros((tokens, width), dtype=torch.bfloat16, device="cuda")
    assert qkv.numel() > 2 ** 31
    c = Case(50, heads, heads, 128, 128, torch.bfloat16)
    qkv[-50:] = c.qkv
    pos = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    pos[-50:] = c.pos
    slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    slots[-50:] = c.slots
    R.qk_norm_rope(qkv, qkv, pos, c.table, heads, heads, 128, **c.kw(), k_cache=c.k, v_cache=c.v, slots=slots)
    c.out.copy_(qkv[-50:])
    c.check()
    assert bool((qkv[:-50] == 0).all())


@gpu
def test_no_tokens():
    c = Case(4, 2, 1, 64, 64, torch.bfloat16)
    out = c.out[:0]
    assert R.qk_norm_rope(c.qkv[:0], out, c.pos[:0], c.table, 2, 1, 64) is out


def test_table():
    t = R.rotary_table(100000, 64, theta=500000.0)
    assert t.shape == (100000, 64) and t.dtype == torch.float32
    for pos, i in ((0, 0), (1, 0), (99999, 0), (99999, 31), (54321, 17)):
        a = pos * 500000.0 ** (-i / 32)
        assert abs(t[pos, i].item() - math.cos(a)) <= 2.0 ** -24 and abs(t[pos, 32 + i].item() - math.sin(a)) <= 2.0 ** -24
    # linear: position 8 of the scaled table is position 2 of the plain one
    assert torch.equal(R.rotary_table(9, 32, scaling="linear", factor=4.0)[8], R.rotary_table(9, 32)[2])
    # theta: the fastest pair turns as before, the slowest `factor` times slower
    plain, wide = R.rotary_table(9, 32), R.rotary_table(9, 32, scaling="theta", factor=4.0)
    assert torch.equal(wide[:, 0], plain[:, 0])
    slow = 10000.0 ** (-15 / 16)
    assert abs(wide[8, 31].item() - math.sin(8 * slow / 4)) <= 2.0 ** -24
    # parts: fast pairs as before, slow ones `factor` times slower, mixed in between
    parts = R.rotary_table(2, 128, scaling="parts", factor=8.0, original_positions=4096)
    for i in range(64):
        speed = 10000.0 ** (-i / 64)
        turns = 4096 * speed / (2 * math.pi)
        kept = min(1.0, max(0.0, (turns - 1) / 31))
        assert abs(parts[1, 64 + i].item() - math.sin(speed * kept + speed * (1 - kept) / 8)) <= 2.0 ** -24
    assert 0 < sum(1 < 4096 * 10000.0 ** (-i / 64) / (2 * math.pi) < 32 for i in range(64)) < 64


def test_refusals():
    c = Case(6, 2, 1, 64, 32, torch.bfloat16, device="cpu")

    def call(qkv=c.qkv, out=c.out, pos=c.pos, table=c.table, heads=2, kv=1, dim=64, **kw):
        R.qk_norm_rope(qkv, out, pos, table, heads, kv, dim, **kw)
    with pytest.raises(TypeError):
        call(qkv=c.qkv.float())
    with pytest.raises(TypeError):
        call(k_cache=c.k.half(), v_cache=c.v.half(), slots=c.slots)
    other = c.v.transpose(1, 2).contiguous().transpose(1, 2)
    for bad in (dict(heads=3), dict(dim=32), dict(dim=24), dict(pos=c.pos.long()), dict(pos=c.pos[:5]), dict(table=c.table.double()),
                dict(table=c.table[:, :24]), dict(table=torch.zeros(500, 80)), dict(q_weight=torch.ones(64)),
                dict(k_weight=torch.ones(32, dtype=torch.bfloat16)), dict(out=c.out[:, :128]), dict(out=c.out[:, :64]),
                dict(k_cache=c.k), dict(k_cache=c.k, v_cache=c.v), dict(k_cache=c.k[:, :, :, :32], v_cache=c.v[:, :, :, :32], slots=c.slots),
                dict(k_cache=c.k, v_cache=other, slots=c.slots), dict(**{**c.cache(), "slots": c.slots.long()})):
        with pytest.raises(ValueError):
            call(**bad)
    wide = torch.zeros((6, 600), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share no memory"):
        call(qkv=wide[:, :256], out=wide[:, 8:264])
    with pytest.raises(ValueError, match="CUDA device"):
        call(qkv=wide[:, :256], out=wide[:, 256:512])       # columns of one matrix, apart
    with pytest.raises(ValueError, match="CUDA device"):
        call()
    for bad in (dict(positions=0), dict(rotary_dim=24), dict(theta=0.0), dict(factor=-1.0), dict(scaling="cubic"),
                dict(scaling="parts", factor=2.0)):
        with pytest.raises(ValueError):
            R.rotary_table(**{**dict(positions=4, rotary_dim=32), **bad})


def test_one_token_in_place_whatever_its_strides():
    """Along one row a stride says nothing."""
    c = Case(1, 2, 1, 32, 16, torch.bfloat16, device="cpu")
    over = torch.as_strided(c.qkv, c.qkv.shape, (0, 1))
    for out in (over, over[:, :64]):
        with pytest.raises(ValueError, match="CUDA device"):
            R.qk_norm_rope(c.qkv, out, c.pos, c.table, 2, 1, 32, **c.kw(), **c.cache())


def test_a_status_that_is_no_block_is_refused():
    """A record has 32 bytes; what is smaller, strided or misaligned would be written past."""
    c = Case(3, 2, 1, 32, 16, torch.bfloat16, device="cpu")
    memory = torch.zeros(17, dtype=torch.int32)
    for bad in (memory[:1], memory[:7], memory[1:], memory[::2][:8]):
        with pytest.raises(ValueError, match="status"):
            R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 2, 1, 32, status=bad, **c.kw())
    with pytest.raises(ValueError, match="CUDA device"):
        R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 2, 1, 32, status=memory[:8], **c.kw())


@gpu
def test_refusals_of_the_native_entry():
    c = Case(6, 2, 1, 64, 32, torch.bfloat16)
    with pytest.raises(RuntimeError, match="power of two"):
        R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 2, 1, 64, k_cache=c.k[:, :12], v_cache=c.v[:, :12], slots=c.slots)
    wide = torch.zeros((6, 600), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="16 bytes"):
        R.qk_norm_rope(wide[:, 4:260], wide[:, 264:520], c.pos, c.table, 2, 1, 64)


def _native_answer(qkv, out, heads, kv, dim, positions, slots, k, v, table, weights=(0, 0)):
    """What the native entry says to a call; those it does not refuse find no device here.  (Tests without a device alone.)"""
    out_heads = heads + kv if out.data_ptr() == qkv.data_ptr() and out.shape == qkv.shape else out.shape[1] // dim
    pages, size = k.shape[:2]
    lib = _native.kernels()
    rc = _native.entry("iris_k_qk_norm_rope")(R._ARGS.pack(
        qkv.data_ptr(), out.data_ptr(), positions.data_ptr(), table.data_ptr(), *weights, k.data_ptr(), v.data_ptr(),
        slots.data_ptr(), 0, 0, qkv.stride(0), out.stride(0), table.stride(0), *k.stride()[:3], out_heads, *table.shape, 0,
        pages, size, qkv.shape[0], heads, kv, dim, 0, 1e-6))
    assert rc < 0
    lib.iris_rotary_last_error.restype = ctypes.c_char_p
    return lib.iris_rotary_last_error().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are not refused must find no device")
def test_memory_that_tokens_or_arguments_share_is_refused():
    """Rows of the cache that meet, whatever pitch they meet by; keys over a part of the values; a cache in qkv or out; positions,
    slots, weights or the table under what is written.  Column blocks side by side, and pages of keys and values in turn, are fine."""
    tokens, heads, kv, dim, pages, size = 6, 2, 2, 64, 3, 4
    big = torch.zeros(1 << 16, dtype=torch.bfloat16)
    qkv, out = big[:6 * 400].view(6, 400)[:, :384], big[4096:4096 + 6 * 384].view(6, 384)
    cache = big[8192:8192 + 2 * pages * size * kv * dim].view(2, pages, size, kv, dim)
    positions, slots = torch.zeros(6, dtype=torch.int32), torch.arange(6, dtype=torch.int32)
    table = torch.zeros(10, 32)
    ok = dict(qkv=qkv, out=out, heads=heads, kv=kv, dim=dim, positions=positions, slots=slots, k=cache[0], v=cache[1], table=table)

    def at(offset, pitches, shape=(pages, size, kv, dim)):
        return torch.as_strided(big, shape, (*pitches, 1), offset)
    turns, columns = big[16384:16384 + 2 * pages * size * kv * dim], big[24576:24576 + 2 * pages * size * kv * dim]
    turns, columns = turns.view(pages, 2, size, kv, dim), columns.view(pages, size, kv, 2 * dim)
    by_head = big[8192:8192 + 2 * pages * size * kv * dim].view(2, pages, kv, size, dim).transpose(2, 3)
    for fine in (dict(), dict(k=turns[:, 0], v=turns[:, 1]), dict(k=columns[..., :dim], v=columns[..., dim:]), dict(out=qkv),
                 dict(out=qkv[:, :128]), dict(k=by_head[0], v=by_head[1]), dict(positions=big[392:404].view(torch.int32)[:6]),
                 dict(k=at(30000, (4096, 64, 512)), v=at(30000 + 256, (4096, 64, 512)))):
        assert "launch" in _native_answer(**{**ok, **fine}), fine
    ints = lambda o: big[o:o + 12].view(torch.int32)   # noqa: E731
    for what, bad in (
            ("overlap", dict(k=at(30000, (1024, 64, 64)), v=at(50000, (1024, 64, 64)))),       # slots and heads at one pitch
            ("overlap", dict(k=at(30000, (64, 64, 512)), v=at(50000, (64, 64, 512)))),         # pages and slots
            ("overlap", dict(k=at(30000, (256, 128, 64)), v=at(50000, (256, 128, 64)))),       # a page shorter than its slots
            ("overlap", dict(v=cache[0])), ("overlap", dict(k=at(30000, (1024, 256, 128)), v=at(30064 - 8, (1024, 256, 128)))),
            ("overlap", dict(v=at(8192 + 512, (512, 128, 64)))),                                # keys' page 1 on
            ("overlap", dict(out=out[:1].expand(6, -1))),
            ("qkv or out", dict(k=at(0, (512, 128, 64)), v=at(40000, (512, 128, 64)))),
            ("qkv or out", dict(k=at(40000, (512, 128, 64)), v=at(4096, (512, 128, 64)))),
            ("positions", dict(positions=ints(4096 + 8))), ("positions", dict(slots=ints(8192 + 64))),
            ("positions", dict(positions=ints(8192 + 1536 + 8))), ("positions", dict(weights=(out.data_ptr() + 128, 0))),
            ("positions", dict(table=big[4096:4096 + 640].view(torch.float32).view(10, 32)))):
        assert what in _native_answer(**{**ok, **bad}), (what, bad)


@gpu
def test_caches_that_overlap_are_refused():
    """Keys and values in one place, or pages that are all one page: two tokens would write to one address."""
    c = Case(6, 2, 1, 64, 32, torch.bfloat16)
    before = c.k.clone()
    with pytest.raises(RuntimeError, match="overlap"):
        R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 2, 1, 64, k_cache=c.k, v_cache=c.k, slots=c.slots)
    one_k, one_v = (t[:1].expand(4, -1, -1, -1) for t in (c.k, c.v))
    with pytest.raises(RuntimeError, match="overlap"):
        R.qk_norm_rope(c.qkv, c.out, c.pos, c.table, 2, 1, 64, k_cache=one_k, v_cache=one_v, slots=c.slots)
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(c.k.float()), torch.nan_to_num(before.float()))
