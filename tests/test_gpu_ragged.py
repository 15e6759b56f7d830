"""The ragged operators against plain implementations in 64 bits (GPU).

Tolerance of the attention, from the arithmetic of the kernels.  With u = 2^-24 (fp32) and
for one output row, S = max over its tokens of scale * sum_d |q_d k_d| bounds every partial sum
of a logit.  A logit is a sum of D products: D additions, each off by at most 2 u S (tensor
cores may truncate instead of round), then two products (scale, log2 e) and the subtraction of
the maximum, each off by at most u times a number of at most 2 S log2 e.  So a weight is off
relatively by at most
    e_w = (2 D + 8) u S + 2^-22 (the hardware's 2^x) + r_p,
where r_p is the rounding of the weights for the tensor cores: they go in as a sum of two
16-bit numbers, each rounded by at most half a step h (bf16 2^-8, fp16 2^-11), so r_p = h^2.
The weighted sum and the weights' sum add N numbers in fp32: N 2 u each at most, and joining
parts multiplies by further 2^x, of which there are at most a handful (16 u allowed).  Hence
    |out - exact| <= (2 e_w + 4 N u + 2^-20) A + h |exact|,  A = sum w |v| / sum w,
    |lse - exact| <= e_w + 2 N u + 2^-20 + 4 u |exact|.
"""

import math

import pytest
import torch

import razorkv_b200 as R
from razorkv_b200 import _lib
from razorkv_b200._lib import DeviceError
from razorkv_b200.kernels import check_device_errors

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool_case(lengths, Hq, Hkv, D, P, dtype, seed, starts=None, layout="hpd", extra=3, nan=True,
               width=None):
    """Pools whose unused rows hold NaN, a shuffled page table whose unused entries are stale
    ids, and queries."""
    g = _gen(seed)
    held = [-(-n // P) for n in lengths]
    slots = sum(held) + extra
    shape = {"hpd": (slots, Hkv, P, D), "phd": (slots, P, Hkv, D)}[layout]
    pools = []
    for _ in range(2):
        t = torch.full(shape, math.nan if nan else 0.0, device="cuda", dtype=dtype)
        pools.append(t if layout == "hpd" else t.transpose(1, 2))
    perm = torch.randperm(slots, generator=g, device="cuda").tolist()
    W = width or max(1, max(held))
    table = torch.randint(0, slots, (len(lengths), W), generator=g, device="cuda")
    at = 0
    for b, (n, h) in enumerate(zip(lengths, held)):
        table[b, :h] = torch.tensor(perm[at: at + h], dtype=torch.int64)
        first = 0 if starts is None else starts[b]
        for pool in pools:
            t = torch.arange(min(first, n), n, device="cuda")
            pool[table[b, t // P], :, t % P] = torch.randn(
                len(t), Hkv, D, generator=g, device="cuda").to(dtype)
        at += h
    q = (torch.randn(len(lengths), Hq, 1, D, generator=g, device="cuda")
         * torch.linspace(0.5, 3, Hq, device="cuda")[:, None, None]).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int64, device="cuda")
    s = None if starts is None else torch.tensor(starts, dtype=torch.int64, device="cuda")
    return q, pools[0], pools[1], table, n, s


def _exact(q, kp, vp, table, lengths, starts, scale=None):
    """(out, lse, bound of out, bound of lse) in 64 bits."""
    B, Hq, _, D = q.shape
    Hkv, P = kp.shape[1:3]
    G = Hq // Hkv
    scale = scale or 1 / math.sqrt(D)
    out = torch.zeros(B, Hq, 1, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    h16 = HALF[q.dtype] if q.dtype != torch.float32 else 0.0
    for b in range(B):
        n = int(lengths[b])
        first = 0 if starts is None else int(starts[b])
        if n <= first:
            continue
        t = torch.arange(first, n, device=q.device)
        k = kp[table[b, t // P], :, t % P].double()     # [N, Hkv, D]
        v = vp[table[b, t // P], :, t % P].double()
        qb = q[b, :, 0].double().view(Hkv, G, D)
        s = torch.einsum("hgd,thd->hgt", qb, k) * scale
        big = torch.einsum("hgd,thd->hgt", qb.abs(), k.abs()).amax(-1) * scale
        w = torch.softmax(s, -1)
        e_w = (2 * D + 8) * U * big + 2.0 ** -22 + h16 * h16
        N = n - first
        o = torch.einsum("hgt,thd->hgd", w, v)
        A = torch.einsum("hgt,thd->hgd", w, v.abs())
        out[b, :, 0] = o.reshape(Hq, D)
        lse[b] = torch.logsumexp(s, -1).reshape(Hq)
        tol[b, :, 0] = ((2 * e_w + 4 * N * U + 2.0 ** -20)[..., None] * A
                        + HALF[q.dtype] * o.abs()).reshape(Hq, D)
        tol_lse[b] = (e_w + 2 * N * U + 2.0 ** -20).reshape(Hq) + 4 * U * lse[b].abs()
    return out, lse, tol, tol_lse


def _compare(case, scale=None, **kwargs):
    q, kp, vp, table, n, s = case
    got, lse = R.ragged_decode_attention(q, kp, vp, table, n, scale=scale, starts=s,
                                         return_lse=True, **kwargs)
    out, ls, tol, tol_lse = _exact(*case, scale=scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    assert lse.dtype == torch.float32 and lse.shape == q.shape[:2]
    off = (got.double() - out).abs()
    # the smallest subnormal of fp16 output rounds by an absolute step
    floor = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    assert bool((off <= tol + floor).all()), float((off / (tol + 1e-30)).max())
    empty = torch.isinf(ls)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    assert bool((((lse.double() - ls).abs() <= tol_lse) | empty).all())
    assert bool((got[empty] == 0).all())
    return got, lse


ODD = [0, 1, 2, 15, 16, 17, 31, 33, 64, 127, 300, 5, 777]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,P", [
    (8, 2, 128, 16), (32, 8, 128, 16), (28, 4, 128, 16), (4, 4, 64, 16), (6, 2, 64, 5),
    (16, 2, 128, 32), (16, 1, 64, 64), (12, 1, 128, 8), (34, 2, 64, 16), (2, 1, 256, 16),
    (10, 2, 96, 16), (5, 5, 80, 16), (3, 1, 20, 7), (4, 2, 17, 1), (8, 1, 32, 128), (40, 1, 256, 3),
    (1, 1, 1, 1), (6, 3, 192, 24), (9, 1, 40, 16)])
def test_attention_shapes(dtype, Hq, Hkv, D, P):
    _compare(_pool_case(ODD, Hq, Hkv, D, P, dtype, seed=Hq * D + P))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lengths", [[1], [0], [0, 0, 0], [16], [2049], [4999, 1], [1, 9001, 0, 3],
                                     [1] * 700, [3] * 129 + [0] * 130, [40000]])
def test_attention_lengths(dtype, lengths):
    _compare(_pool_case(lengths, 8, 2, 64, 16, dtype, seed=sum(lengths) % 97))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("P", [5, 16, 64])
def test_attention_starts(dtype, P):
    lengths = [100, 100, 100, 33, 0, 1, 2000, 2000, 50, 16, 17]
    starts = [0, 99, 100, 17, 5, 0, 1999, 1001, 1 << 40, 15, 16]
    _compare(_pool_case(lengths, 8, 2, 128, P, dtype, seed=P, starts=starts))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_attention_layouts(dtype):
    """Token-major pools, strided and misaligned queries and outputs, a wider table, a scale."""
    case = _pool_case(ODD, 8, 2, 128, 16, dtype, seed=1, layout="phd", width=60)
    base, _ = _compare(case)
    _compare(case, scale=0.3)
    q, kp, vp, table, n, s = case
    B, Hq, _, D = q.shape
    wide = torch.randn(B, 1, Hq, D + 24, device="cuda").to(dtype)
    qs = wide[..., 8: 8 + D].transpose(1, 2)
    qs.copy_(q)
    assert torch.equal(R.ragged_decode_attention(qs, kp, vp, table, n), base)
    qs = wide[..., 3: 3 + D].transpose(1, 2)         # rows off every vector boundary
    qs.copy_(q)
    _compare((qs, kp, vp, table, n, s))
    _compare((qs, kp, vp, table, n, s), out=torch.empty_like(wide)[..., 1: 1 + D].transpose(1, 2))
    big = torch.empty(B, 2 * Hq, 1, 2 * D, device="cuda", dtype=dtype).fill_(7)
    _compare(case, out=big[:, ::2, :, D:])
    assert bool((big[:, 1::2] == 7).all()) and bool((big[..., :D] == 7).all())
    tw = torch.full((B, 130), -1, dtype=torch.int64, device="cuda")
    tw[:, ::2][:, :60] = table
    _compare((q, kp, vp, tw[:, ::2][:, :60], n, s))
    # pools whose rows are not 16-byte aligned
    off = [torch.full((kp.shape[0], 2, 16, 129), math.nan, device="cuda", dtype=dtype)[..., 1:] for _ in "kv"]
    off[0].copy_(kp), off[1].copy_(vp)
    _compare((q, off[0], off[1], table, n, s))


def test_attention_large_logits():
    """Logits of hundreds: the running maximum has to be taken out before the power."""
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        q, kp, vp, table, n, s = _pool_case([400, 37, 1], 8, 2, 64, 16, dtype, seed=3)
        _compare(((q * 16).to(dtype), kp, vp, table, n, s), scale=1.0)


def test_attention_nan_inside_stays_in_its_request():
    q, kp, vp, table, n, s = _pool_case([50, 70, 90], 4, 2, 128, 16, torch.bfloat16, seed=4)
    clean = R.ragged_decode_attention(q, kp, vp, table, n)
    kp[table[1, 2], 1, 5] = math.nan
    out, lse = R.ragged_decode_attention(q, kp, vp, table, n, return_lse=True)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    assert torch.equal(out[1, :2], clean[1, :2])
    assert bool(torch.isnan(out[1, 2:]).all()) and bool(torch.isnan(lse[1, 2:]).all())


def test_attention_repeats_bit_for_bit_and_shares_pages():
    case = _pool_case([3000, 1, 500, 2222], 28, 4, 128, 16, torch.bfloat16, seed=5)
    first = [t.clone() for t in _compare(case)]
    for _ in range(5):
        again = R.ragged_decode_attention(*case[:5], return_lse=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    q, kp, vp, table, n, s = case
    table[1] = table[0]      # request 1 shares request 0's pages
    n[1] = 1600
    _compare((q, kp, vp, table, n, s))


def test_attention_past_32_bit_offsets():
    """Rows whose element offset is beyond 2^32."""
    P, Hkv, D, dtype = 16, 8, 128, torch.bfloat16
    slots = (1 << 32) // (Hkv * P * D) + 40
    kp = torch.empty(slots, Hkv, P, D, dtype=dtype, device="cuda")
    vp = torch.empty_like(kp)
    g = _gen(6)
    used = torch.tensor([slots - 1, 3, slots - 17, (1 << 31) // (Hkv * P * D) + 1], device="cuda")
    for pool in (kp, vp):
        pool[used] = torch.randn(4, Hkv, P, D, generator=g, device="cuda").to(dtype)
    table = torch.stack([used, used.flip(0)])
    n = torch.tensor([64, 35], device="cuda")
    q = torch.randn(2, 32, 1, D, generator=g, device="cuda").to(dtype)
    _compare((q, kp, vp, table, n, None))
    # the append reaches the same rows
    slot = torch.tensor([int(used[0]) * P + 15, int(used[2]) * P], device="cuda")
    rows = torch.randn(2, Hkv, D, generator=g, device="cuda").to(dtype)
    R.ragged_append(rows, -rows, kp, vp, slot)
    assert torch.equal(kp[used[0], :, 15], rows[0]) and torch.equal(vp[used[2], :, 0], -rows[1])
    check_device_errors()


def test_attention_empty_batch_and_no_columns():
    kp = torch.zeros(2, 2, 16, 64, device="cuda")
    q = torch.zeros(0, 4, 1, 64, device="cuda")
    table = torch.zeros(0, 3, dtype=torch.int64, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    out, lse = R.ragged_decode_attention(q, kp, kp, table, none, return_lse=True)
    assert out.shape == (0, 4, 1, 64) and lse.shape == (0, 4)
    q = torch.ones(3, 4, 1, 64, device="cuda")
    table = torch.zeros(3, 0, dtype=torch.int64, device="cuda")
    out, lse = R.ragged_decode_attention(q, kp, kp, table, torch.zeros(3, dtype=torch.int64, device="cuda"),
                                         return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_attention_device_errors():
    check_device_errors()
    q, kp, vp, table, n, s = _pool_case([40, 70], 8, 2, 128, 16, torch.bfloat16, seed=7, nan=False)
    bad = table.clone()
    bad[1, 1], bad[1, 2] = kp.shape[0], -5
    out = R.ragged_decode_attention(q, kp, vp, bad, n)
    with pytest.raises(DeviceError) as e:
        check_device_errors()
    assert e.value.code == 2
    check_device_errors()
    read = bad.clone()
    read[1, 1:3] = 0
    assert torch.equal(out, R.ragged_decode_attention(q, kp, vp, read, n))
    full = torch.tensor([-3, table.shape[1] * 16 + 1], device="cuda")
    out = R.ragged_decode_attention(q, kp, vp, table, full)
    with pytest.raises(DeviceError) as e:
        check_device_errors(q.device)
    assert e.value.code == 3
    bound = torch.tensor([0, table.shape[1] * 16], device="cuda")
    assert torch.equal(out, R.ragged_decode_attention(q, kp, vp, table, bound))
    with pytest.raises(IndexError):
        R.ragged_decode_attention(q, kp, vp, table, full, validate=True)
    with pytest.raises(IndexError):
        R.ragged_decode_attention(q, kp, vp, bad, n, validate=True)
    check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (16, 1, 128), (12, 3, 64), (6, 2, 200), (3, 1, 33)])
@pytest.mark.parametrize("lengths", [[256], [129, 1, 0, 65], [250] * 9, [17, 64, 33, 100, 32, 256, 255],
                                     [128, 120, 113, 40, 16]])
def test_attention_tables_of_few_tiles(dtype, Hq, Hkv, D, lengths):
    # tables with room for 4 to 33 tiles, from full to a token long, of calls whose segments are few
    P = 32
    for starts in (None, [max(0, n - 37 * (i + 1)) for i, n in enumerate(lengths)]):
        for width in (-(-max(lengths) // P), 8, 9):
            if width * P >= max(lengths):
                _compare(_pool_case(lengths, Hq, Hkv, D, P, dtype, seed=11, starts=starts, width=width))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("width", [200, 32767, 32769])
def test_attention_wide_tables(dtype, width):
    """Tables whose capacity in tiles, or in tokens, is beyond 31 bits."""
    case = _pool_case([70000, 131077, 3] + [0] * 59 + [65536, 1], 2, 1, 8, 65536, dtype, seed=11,
                      width=width)
    _compare(case)
    check_device_errors()


# ---- append -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,Hkv,D,P,layout,offset", [
    (1, 8, 128, 16, "hpd", 0), (64, 8, 128, 16, "hpd", 0), (1003, 3, 64, 5, "phd", 0),
    (77, 2, 20, 7, "hpd", 0), (50, 4, 64, 16, "hpd", 1), (9, 1, 1, 1, "hpd", 0),
    (5000, 2, 256, 32, "hpd", 0), (0, 2, 64, 16, "hpd", 0)])
def test_append(dtype, T, Hkv, D, P, layout, offset):
    g = _gen(T + D)
    slots = -(-T // P) + 4
    shape = (slots, Hkv, P, D + offset) if layout == "hpd" else (slots, P, Hkv, D + offset)
    pools = [torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in "kv"]
    views = [(t if layout == "hpd" else t.transpose(1, 2))[..., offset:] for t in pools]
    key, value = (torch.randn(T, Hkv, D, generator=g, device="cuda").to(dtype) for _ in "kv")
    slot = torch.randperm(slots * P, generator=g, device="cuda")[:T]
    slot[torch.rand(T, generator=g, device="cuda") < 0.2] = -1
    expect = [t.clone() for t in views]
    keep = slot >= 0
    for e, rows in zip(expect, (key, value)):
        e[slot[keep] // P, :, slot[keep] % P] = rows[keep]
    R.ragged_append(key, value, views[0], views[1], slot)
    assert torch.equal(views[0], expect[0]) and torch.equal(views[1], expect[1])
    # rows as a projection leaves them, [T, heads of q, k and v, D] in one tensor, and a
    # strided slot map
    joint = torch.randn(max(T, 1), 3 * Hkv, D, generator=g, device="cuda").to(dtype)[:T]
    two = torch.stack([slot, slot], 1)[:, 0]
    k, v = joint[:, Hkv: 2 * Hkv], joint[:, 2 * Hkv:]
    for e, rows in zip(expect, (k, v)):
        e[slot[keep] // P, :, slot[keep] % P] = rows[keep]
    R.ragged_append(k, v, views[0], views[1], two)
    assert torch.equal(views[0], expect[0]) and torch.equal(views[1], expect[1])
    check_device_errors()


def test_append_skips_slots_past_the_pool():
    check_device_errors()
    kp = torch.zeros(4, 2, 16, 64, device="cuda")
    vp = torch.zeros_like(kp)
    rows = torch.ones(4, 2, 64, device="cuda")
    slot = torch.tensor([64, 5, -(1 << 62), (1 << 63) - 1], device="cuda")
    R.ragged_append(rows, rows, kp, vp, slot)
    with pytest.raises(DeviceError) as e:
        check_device_errors()
    assert e.value.code == 2
    assert float(kp.sum()) == 128 and float(vp[0, :, 5].sum()) == 128


# ---- page tables ---------------------------------------------------------------------------------
def _plain_tables(lengths, new, table, ring, state, P, most):
    """The definition, one request after another, on lists."""
    table, ring = [list(r) for r in table], list(ring)
    W = len(table[0]) if table else 0
    C, R_ = len(ring), len(lengths)
    head, count, _ = state
    pages = lambda x: -(-x // P)  # noqa: E731
    need = sum(max(0, pages(m) - pages(n)) for n, m in zip(lengths, new))
    give = sum(max(0, pages(n) - pages(m)) for n, m in zip(lengths, new))
    fresh = sum(max(0, m - n) for n, m in zip(lengths, new))
    if (need > count or fresh > most or count - need + give > C or not 0 <= head < C
            or not 0 <= count <= C or any(not 0 <= x <= W * P for x in lengths + new)):
        return lengths, [-1] * most, [0] * most, [0] * (R_ + 1), [head, count, 0], table, ring, False
    slots, positions, starts = [], [], [0]
    tail = head + count
    for r, (n, m) in enumerate(zip(lengths, new)):
        for j in range(pages(n), pages(m)):
            table[r][j] = ring[head % C]
            head += 1
        for t in range(n, m):
            slots.append(table[r][t // P] * P + t % P)
            positions.append(t)
        starts.append(len(slots))
        for j in range(pages(m), pages(n)):
            ring[tail % C] = table[r][j]
            tail += 1
    pad = most - len(slots)
    return (new, slots + [-1] * pad, positions + [0] * pad, starts,
            [head % C, tail - head, 0], table, ring, True)


def _check_tables(lengths, new, table, ring, state, P, most, inplace=False):
    """One call against the definition; returns its RaggedTables."""
    want = _plain_tables(lengths.tolist(), new.tolist(), table.tolist(), ring.tolist(),
                         state.tolist(), P, most)
    before = lengths.clone(), state.clone()
    t = R.ragged_page_tables(lengths, new, table, ring, state, P, most, inplace=inplace)
    assert t.lengths.tolist() == list(want[0])
    assert t.slot_map.tolist() == want[1] and t.positions.tolist() == want[2]
    assert t.token_starts.tolist() == want[3] and t.free_state.tolist() == want[4]
    assert table.tolist() == want[5] and ring.tolist() == want[6]
    if inplace:
        assert t.lengths is lengths and t.free_state is state
    else:
        assert torch.equal(lengths, before[0]) and torch.equal(state, before[1])
    if want[7]:
        check_device_errors()
    else:
        with pytest.raises(DeviceError) as e:
            check_device_errors()
        assert e.value.code == 4
    return t


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("requests,P,W,most", [(1, 16, 8, 40), (7, 1, 30, 100), (64, 5, 40, 3000),
                                               (300, 16, 64, 20000), (2500, 3, 12, 9000)])
def test_tables_over_many_steps(requests, P, W, most, inplace):
    """Steps that grow, admit, retire and shorten; every page stays in one place: a request's
    row or the ring."""
    check_device_errors()
    g = torch.Generator().manual_seed(requests + P)
    slots = requests * W // 2 + 5
    ring, state = R.ragged_free_ring(slots, "cuda")
    table = torch.full((requests, W), -7, dtype=torch.int64, device="cuda")
    n = torch.zeros(requests, dtype=torch.int64, device="cuda")
    refused = 0
    for step in range(12):
        kind = torch.randint(0, 6, (requests,), generator=g).cuda()
        some = torch.randint(0, W * P + 1, (requests,), generator=g).cuda()
        m = torch.where(kind < 3, (n + 1).clamp(max=W * P), n)
        m = torch.where(kind == 3, some, m)
        m = torch.where(kind == 4, 0, m)
        before = n.clone()
        t = _check_tables(n, m, table, ring, state, P, most, inplace)
        n, state = t.lengths, t.free_state
        refused += int(not torch.equal(n, m) and torch.equal(n, before))
        held = (n + P - 1) // P
        pages = table[torch.arange(W, device="cuda")[None] < held[:, None]].tolist()
        head, count = state.tolist()[:2]
        pages += [int(ring[(head + i) % slots]) for i in range(count)]
        assert sorted(pages) == list(range(slots))
    assert refused < 12


def test_tables_repeat_and_corners():
    check_device_errors()
    dev = "cuda"
    ring, state = R.ragged_free_ring(10, dev)
    table = torch.zeros(3, 4, dtype=torch.int64, device=dev)
    n = torch.zeros(3, dtype=torch.int64, device=dev)
    m = torch.tensor([4, 0, 9], device=dev)
    a = _check_tables(n, m, table, ring, state, 4, 13)
    b = _check_tables(n, m, table, ring, state, 4, 13)     # nothing but its inputs counts
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # exactly as many tokens as fit, one too many, no entry at all
    _check_tables(n, m, table, ring, state, 4, 12)
    _check_tables(a.lengths, a.lengths, table, ring, a.free_state, 4, 0)
    _check_tables(a.lengths, torch.zeros_like(n), table, ring, a.free_state, 4, 0)
    # columns of a wider table, and a single row of one
    wide = torch.full((5, 9), 9, dtype=torch.int64, device=dev)
    c = _check_tables(n, m, wide[:3, 2:6], ring, state, 4, 13)
    assert torch.equal(c.slot_map, a.slot_map) and torch.equal(wide[:3, 2:6][0, :1], table[0, :1])
    assert bool((wide[3:] == 9).all()) and bool((wide[:, :2] == 9).all()) and bool((wide[:, 6:] == 9).all())
    _check_tables(n[:1], m[:1], wide[4:5, :4], ring, state, 4, 4)
    # no requests
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    t = _check_tables(none, none, torch.zeros(0, 4, dtype=torch.int64, device=dev), ring, state, 4, 5)
    assert t.token_starts.tolist() == [0] and t.slot_map.tolist() == [-1] * 5
    # a table without columns
    z = torch.zeros(2, dtype=torch.int64, device=dev)
    _check_tables(z, z, torch.zeros(2, 0, dtype=torch.int64, device=dev), ring, state, 4, 5)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("most", [13, 5000])
def test_tables_refusals_change_nothing(inplace, most):
    check_device_errors()
    dev = "cuda"

    def call(n, m, state=(0, 3, 0), most=most):
        ring = torch.arange(10, device=dev)
        table = torch.full((2, 4), 9, dtype=torch.int64, device=dev)
        t = lambda v: torch.tensor(v, dtype=torch.int64, device=dev)  # noqa: E731
        return _check_tables(t(n), t(m), table, ring, t(state), 4, most, inplace)

    call([0, 0], [8, 4])                       # three pages: granted
    call([0, 0], [8, 5])                       # four pages of three
    call([0, 0], [17, 0])                      # past the table
    call([-1, 0], [1, 0])
    call([0, 0], [-1, 0])
    call([0, 17], [0, 17])
    call([0, 1 << 62], [0, 1])
    call([3, 3], [4, 4], most=1)               # more new tokens than entries
    call([0, 0], [1, 1], state=(10, 3, 0))     # a head outside the ring
    call([0, 0], [1, 1], state=(0, 11, 0))
    call([0, 0], [1, 1], state=(-1, 3, 0))
    call([8, 8], [0, 0], state=(5, 7, 0))      # more pages back than the ring holds
    call([8, 8], [0, 4], state=(5, 7, 0))      # exactly as many


def test_tables_pages_outside_the_pool():
    check_device_errors()
    ring = torch.tensor([2, 77, 0], device="cuda")
    table = torch.tensor([[-4, 0], [1, 0]], device="cuda")
    n = torch.tensor([2, 4], device="cuda")
    state = torch.tensor([0, 3, 0], device="cuda")
    t = R.ragged_page_tables(n, torch.tensor([5, 6], device="cuda"), table, ring, state, 4, 6)
    # request 0's page -4 and request 1's new page 77 are no pages of three
    assert t.slot_map.tolist() == [-1, -1, 8, -1, -1, -1]
    with pytest.raises(DeviceError) as e:
        check_device_errors()
    assert e.value.code == 2


# ---- together ---------------------------------------------------------------------------------
def _serve(dtype, captured, P=16, steps=14, Hq=8, Hkv=2, D=64, layers=2, requests=6, seed=0):
    """Requests come, grow and leave; every step's attention against each request's own
    history in 64 bits."""
    g = _gen(seed)
    W, most, slots = 12, 150, 60
    pools = [[torch.full((slots, Hkv, P, D), math.nan, dtype=dtype, device="cuda") for _ in "kv"]
             for _ in range(layers)]
    ring, state = R.ragged_free_ring(slots, "cuda")
    table = torch.zeros(requests, W, dtype=torch.int64, device="cuda")
    n = torch.zeros(requests, dtype=torch.int64, device="cuda")
    m = torch.zeros_like(n)
    key = torch.zeros(layers, most, Hkv, D, dtype=dtype, device="cuda")
    value = torch.zeros_like(key)
    q = torch.zeros(layers, requests, Hq, 1, D, dtype=dtype, device="cuda")
    outs = torch.zeros_like(q)
    lses = torch.zeros(layers, requests, Hq, device="cuda")

    def step():
        t = R.ragged_page_tables(n, m, table, ring, state, P, most, inplace=True)
        for layer in range(layers):
            R.ragged_append(key[layer], value[layer], *pools[layer], t.slot_map)
            _, lse = R.ragged_decode_attention(q[layer], *pools[layer], table, n, return_lse=True,
                                               out=outs[layer])
            lses[layer].copy_(lse)

    graph = None
    if captured:
        step()      # nothing to do yet: every length is zero
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    history = [[torch.zeros(2, 0, Hkv, D, dtype=dtype, device="cuda") for _ in range(requests)]
               for _ in range(layers)]
    have = [0] * requests
    r = torch.Generator().manual_seed(seed)
    for i in range(steps):
        want = []
        for b in range(requests):
            u = float(torch.rand(1, generator=r))
            if have[b] == 0:
                want.append(int(torch.randint(1, 40, (1,), generator=r)) if u < 0.6 else 0)
            else:
                want.append(0 if u < 0.15 else have[b] + 1)
        m.copy_(torch.tensor(want))
        key.copy_(torch.randn(key.shape, generator=g, device="cuda"))
        value.copy_(torch.randn(value.shape, generator=g, device="cuda"))
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        at = 0
        for b in range(requests):
            new = max(0, want[b] - have[b])
            for layer in range(layers):
                old = history[layer][b][:, : min(have[b], want[b])]
                rows = torch.stack([key[layer, at: at + new], value[layer, at: at + new]])
                history[layer][b] = torch.cat([old, rows], 1)
            at += new
        graph.replay() if captured else step()
        assert n.tolist() == want
        for layer in range(layers):
            h = history[layer]
            # each request's history as a pool of one page
            long = max(1, max(want))
            kp = torch.zeros(requests, Hkv, long, D, dtype=dtype, device="cuda")
            vp = torch.zeros_like(kp)
            for b in range(requests):
                kp[b, :, : want[b]] = h[b][0].transpose(0, 1)
                vp[b, :, : want[b]] = h[b][1].transpose(0, 1)
            ids = torch.arange(requests, device="cuda")[:, None]
            out, lse, tol, tol_lse = _exact(q[layer], kp, vp, ids, n, None)
            assert bool(((outs[layer].double() - out).abs() <= tol + 2.0 ** -25).all())
            fine = torch.isfinite(lse)
            assert torch.equal(fine, torch.isfinite(lses[layer]))
            assert bool((((lses[layer].double() - lse).abs() <= tol_lse) | ~fine).all())
        have = want
    check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(dtype, captured):
    _serve(dtype, captured, P=16 if dtype != torch.float32 else 5, seed=8)


def test_two_graphs_on_two_streams():
    """Graphs captured on one stream and replayed at the same time on two do not share
    scratch memory."""
    cases = [_pool_case([n, 3 * n], 8, 2, 128, 16, torch.bfloat16, seed=n) for n in (1500, 900)]
    want = [R.ragged_decode_attention(*c[:5], return_lse=True) for c in cases]
    graphs, got = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(R.ragged_decode_attention(*c[:5], return_lse=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (a, b), (x, y) in zip(want, got):
        assert torch.equal(a, x) and torch.equal(b, y)


def test_side_streams_at_the_same_time():
    cases = [_pool_case([n, n // 2], 16, 4, 64, 16, torch.float16, seed=n) for n in (700, 2000, 5000)]
    want = [R.ragged_decode_attention(*c[:5]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(R.ragged_decode_attention(*c[:5]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_torch_ops():
    q, kp, vp, table, n, s = _pool_case([40, 3], 8, 2, 64, 16, torch.float16, seed=9)
    out, lse = torch.ops.razorkv.ragged_decode_attention(q, kp, vp, table, n)
    a, b = R.ragged_decode_attention(q, kp, vp, table, n, return_lse=True)
    assert torch.equal(out, a) and torch.equal(lse, b)
    out, _ = torch.ops.razorkv.ragged_decode_attention(q, kp, vp, table, n, 0.5, n - 2)
    assert torch.equal(out, R.ragged_decode_attention(q, kp, vp, table, n, 0.5, n - 2))
    rows = torch.ones(1, 2, 64, device="cuda", dtype=torch.float16)
    torch.ops.razorkv.ragged_append(rows, rows, kp, vp, torch.tensor([17], device="cuda"))
    assert bool((kp[1, :, 1] == 1).all())
    ring, state = R.ragged_free_ring(4, "cuda")
    t = torch.zeros(1, 4, dtype=torch.int64, device="cuda")
    z = torch.zeros(1, dtype=torch.int64, device="cuda")
    got = torch.ops.razorkv.ragged_page_tables(z, z + 3, t, ring, state, 2, 4)
    assert got[1].tolist() == [0, 1, 2, -1] and got[4].tolist() == [2, 2, 0]
    meta = torch.ops.razorkv.ragged_decode_attention(*(x.to("meta") for x in (q, kp, vp, table, n)))
    assert meta[0].shape == out.shape and meta[1].shape == lse.shape


def test_launches_are_counted():
    lib = _lib.load()
    q, kp, vp, table, n, s = _pool_case([40, 3], 8, 2, 64, 16, torch.float16, seed=10)
    before = lib.rkv_launch_count()
    R.ragged_decode_attention(q, kp, vp, table, n)
    assert lib.rkv_launch_count() > before


@pytest.mark.parametrize("dtype,Hq,Hkv,D,P,lengths", [
    (torch.bfloat16, 32, 8, 128, 16, [30011, 5, 0, 17000, 64, 9000]),
    (torch.float16, 28, 4, 128, 16, [90001, 1, 33]),
    (torch.bfloat16, 16, 16, 64, 16, [20000, 20001, 7, 19999]),
    (torch.float16, 32, 2, 128, 64, [60000, 300, 41000]),
    (torch.bfloat16, 12, 4, 256, 5, [20000, 15, 20003]),
    (torch.float32, 8, 4, 128, 16, [20000, 3, 30001]),
])
def test_attention_large(dtype, Hq, Hkv, D, P, lengths):
    """Long requests beside short ones; they repeat bit for bit, and as a graph whose lengths change."""
    case = _pool_case(lengths, Hq, Hkv, D, P, dtype, seed=sum(lengths))
    out, lse = (t.clone() for t in _compare(case))
    q, kp, vp, table, n, s = case
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again = R.ragged_decode_attention(q, kp, vp, table, n, return_lse=True)
    for _ in range(5):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    # the same tables with little in them
    few = torch.tensor([min(x, 40 + 3 * i) for i, x in enumerate(lengths)], device="cuda")
    _compare((q, kp, vp, table, few, s))
    n.copy_(few)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(again[0], R.ragged_decode_attention(q, kp, vp, table, few))
    check_device_errors()
