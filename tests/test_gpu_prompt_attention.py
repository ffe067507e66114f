"""GPU prompt attention against plain attention in 64 bits, within bounds that follow from its roundings (_attention16)."""

from __future__ import annotations

import pytest
import torch

from _attention16 import assert_within, attention64, offsets, packed_attention64
from _helpers import require_gpu

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _op(q, k, v, cu_q, *, scale=None, cu_k=None, heads=None):
    from prism_infer.ops.prompt_attention import prompt_attention

    cu = torch.tensor(cu_q, dtype=torch.int32, device="cuda")
    ck = None if cu_k is None else torch.tensor(cu_k, dtype=torch.int32, device="cuda")
    return prompt_attention(q, k, v, cu, num_heads=q.shape[1], num_kv_heads=k.shape[1],
                            scale=q.shape[2] ** -0.5 if scale is None else scale, cu_seqlens_k=ck)


def _inputs(seed, tokens_q, tokens_k, heads, kv_heads, dim, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens_q, heads, dim, generator=g).to(dtype),
            torch.randn(tokens_k, kv_heads, dim, generator=g).to(dtype),
            torch.randn(tokens_k, kv_heads, dim, generator=g).to(dtype))


def _check(q, k, v, cu_q, cu_k=None, label="", scale=None):
    got = _op(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k=cu_k, scale=scale)
    want, bound = packed_attention64(q, k, v, cu_q, cu_q if cu_k is None else cu_k,
                                     q.shape[2] ** -0.5 if scale is None else scale)
    assert_within(got, want, bound, label)
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (8, 8, 128), (16, 2, 64), (6, 2, 128), (5, 1, 64), (16, 1, 128),
                                                (1, 1, 64)])
def test_lengths_heads_dims(heads, kv_heads, dim, dtype):
    require_gpu()
    lens = [1, 17, 0, 64, 65, 31, 32, 33, 130, 300]
    cu = offsets(lens)
    _check(*_inputs(heads * 100 + dim, cu[-1], cu[-1], heads, kv_heads, dim, dtype), cu, label=f"{heads}/{kv_heads}/{dim}")


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_queries_behind_and_before_their_keys(dtype, dim):
    """More keys than queries; fewer, so that the first rows see nothing; no keys; no queries."""

    require_gpu()
    lq, lk = [5, 40, 70, 1, 9, 0, 200], [300, 10, 70, 1000, 0, 33, 199]
    cu_q, cu_k = offsets(lq), offsets(lk)
    got = _check(*_inputs(7, cu_q[-1], cu_k[-1], 8, 2, dim, dtype), cu_q, cu_k)
    assert (got[cu_q[1]:cu_q[1] + 30] == 0).all() and (got[cu_q[4]:cu_q[5]] == 0).all()


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 64)])
@pytest.mark.parametrize("batch,heads,kv_heads,longest", [(1, 8, 2, 6000), (5, 8, 1, 3000), (70, 4, 1, 1500), (255, 2, 1, 700)])
def test_keys_split_over_workgroups(batch, heads, kv_heads, longest, dtype, dim):
    """Few rows behind many keys, some behind few: blocks of many parts and of one, rows outside, rows without a key."""

    require_gpu()
    g = torch.Generator().manual_seed(batch)
    lq = torch.randint(0, 4, (batch,), generator=g).tolist()
    lk = torch.randint(0, longest, (batch,), generator=g).tolist()
    lk[-1] = 2
    lq[0], lk[0] = 3, longest
    cu_q, cu_k = offsets(lq, start=2), offsets(lk, start=1)
    q, k, v = _inputs(batch + 1, cu_q[-1] + 5, cu_k[-1] + 3, heads, kv_heads, dim, dtype)
    got = _check(q, k, v, cu_q, cu_k)
    assert (got[:2] == 0).all() and (got[cu_q[-1]:] == 0).all()
    # values that are no numbers, in a part that others do not see
    v[cu_k[1] - 1, 0, 3] = float("nan")
    v[cu_k[0] + 40, 0, 5] = float("inf")
    _check(q, k, v, cu_q, cu_k)


# few long sequences whose blocks are about as many as the CUs of a chip with 256: (query lengths, more keys, heads, kv heads)
WIDE = [([1000], [0], 32, 8, 128), ([600, 520], [400, 180], 32, 8, 128), ([1001], [0], 20, 20, 64), ([2040, 7], [9, 0], 16, 16, 64),
        ([200, 200, 112], [2800, 700, 288], 32, 8, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,more,heads,kv_heads,dim", WIDE)
def test_as_many_blocks_as_cus(lq, more, heads, kv_heads, dim, dtype):
    require_gpu()
    lk = [n + m for n, m in zip(lq, more)]
    cu_q, cu_k = offsets(lq, 3), offsets(lk, 5)
    q, k, v = _inputs(25 + dim, cu_q[-1] + 2, cu_k[-1] + 1, heads, kv_heads, dim, dtype)
    want, bound = packed_attention64(q, k, v, cu_q, cu_k, dim ** -0.5)
    k[:5] = k[-1:] = v[:5] = v[-1:] = float("nan")
    assert_within(_op(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k=cu_k), want, bound)


@pytest.mark.parametrize("what", ["nan", "-inf"])
def test_no_numbers_where_blocks_are_as_many_as_cus(what):
    require_gpu()
    q, k, v = _inputs(26, 1001, 1001, 20, 20, 64, BF16)
    v[300, 2, 5] = v[850, 7, 60] = float(what)
    want, bound = attention64(q, k, v, 0.125)
    assert not want.isfinite().all()
    assert_within(_op(q.cuda(), k.cuda(), v.cuda(), [0, 1001]), want, bound)


def test_split_is_the_same_in_a_captured_graph():
    require_gpu()
    from prism_infer.ops.prompt_attention import prompt_attention

    q, k, v = (x.cuda() for x in _inputs(21, 12, 9000, 8, 2, 128, BF16))
    cu_q = torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda")
    cu_k = torch.tensor([0, 6000, 9000], dtype=torch.int32, device="cuda")

    def call():
        return prompt_attention(q, k, v, cu_q, num_heads=8, num_kv_heads=2, scale=0.1, cu_seqlens_k=cu_k)

    call()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second = call(), call()
    with torch.cuda.graph(other):
        third = call()
    for offs in ([0, 6000, 9000], [0, 4, 9000], [0, 9000, 9000], [0, 50, 80]):
        cu_k.copy_(torch.tensor(offs, dtype=torch.int32))
        graph.replay()
        other.replay()
        want = call()
        assert torch.equal(first, want) and torch.equal(second, want) and torch.equal(third, want), offs


def test_many_short_sequences():
    require_gpu()
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 40, (150,), generator=g).tolist()
    cu = offsets(lens)
    _check(*_inputs(4, cu[-1], cu[-1], 8, 2, 128, BF16), cu)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_with_rising_and_falling_scores(dtype):
    """Scores that rise along the keys raise the running max again and again; the last rows see 2500 keys."""

    require_gpu()
    n = 2500
    q, k, v = _inputs(11, n, n, 4, 1, 128, dtype)
    ramp = torch.linspace(-2, 2, n)[:, None]
    q[:, 0] = 1.0
    k[:, 0] = (0.3 * k[:, 0].float() + ramp).to(dtype)       # head 0: up to |score| 22
    q[:, 1] = -1.0                                           # head 1: the first keys are the largest
    _check(q, k, v, [0, n])


def test_scales_of_either_sign_and_zero():
    require_gpu()
    cu = [0, 90, 140]
    q, k, v = _inputs(12, 140, 140, 4, 2, 128, BF16)
    for scale in (0.0, -0.2, 1.0):
        _check(q, k, v, cu, scale=scale, label=f"scale {scale}")


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 128), (BF16, 64)])
def test_rows_outside_the_sequences_are_zero(dtype, dim):
    require_gpu()
    cu = offsets([30, 77, 4], start=9)
    q, k, v = _inputs(13, 400, 400, 8, 4, dim, dtype)
    torch.full((400 * 8 * dim,), float("nan"), dtype=dtype, device="cuda")  # (freed: the output may get this memory)
    got = _check(q, k, v, cu)
    assert (got[:9] == 0).all() and (got[cu[-1]:] == 0).all()
    assert (_op(q.cuda(), k.cuda(), v.cuda(), [0]) == 0).all()  # no sequence at all


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_layouts(dtype):
    """Views of a packed projection, heads before tokens, shared (expanded) values, rows off their 16 bytes, one token."""

    require_gpu()
    cu, n, heads, kv, dim = [0, 70, 101], 101, 8, 2, 128
    g = torch.Generator().manual_seed(14)
    wide = torch.randn(n, (heads + 2 * kv) * dim, generator=g).to(dtype).cuda()
    q, k, v = (x.unflatten(1, (-1, dim)) for x in wide.split([heads * dim, kv * dim, kv * dim], dim=1))
    want, bound = packed_attention64(q.cpu(), k.cpu(), v.cpu(), cu, cu, dim ** -0.5)
    assert_within(_op(q, k, v, cu), want, bound, "packed projection")
    by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert_within(_op(*by_head, cu), want, bound, "heads first")
    odd = [torch.empty(n, x.shape[1], dim + 1, dtype=dtype, device="cuda")[..., 1:].copy_(x) for x in (q, k, v)]
    assert_within(_op(*odd, cu), want, bound, "rows off their 16 bytes")
    columns = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert_within(_op(*columns, cu), want, bound, "dims not contiguous")
    one = v[:, :1].expand(n, kv, dim)
    want, bound = packed_attention64(q.cpu(), k.cpu(), one.cpu(), cu, cu, dim ** -0.5)
    assert_within(_op(q, k, one, cu), want, bound, "expanded values")
    single = torch.empty(1, heads * dim + 3, dtype=dtype, device="cuda")[:, :heads * dim].copy_(wide[:1, :heads * dim])
    want, bound = attention64(q[:1].cpu(), k[:1].cpu(), v[:1].cpu(), dim ** -0.5)
    assert_within(_op(single.view(1, heads, dim), k[:1], v[:1], [0, 1]), want, bound, "one token, odd stride")


@pytest.mark.parametrize("what", ["nan", "inf", "-inf", "both"])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(dtype, dim, what):
    require_gpu()
    cu = [0, 200, 290]
    q, k, v = _inputs(15, 290, 290, 8, 2, dim, dtype)
    special = float("nan" if what == "both" else what)
    v[150, 1, 5] = special     # in the middle of a tile: rows 0..149 do not see it
    v[199, 0, 0] = special     # the last key of a sequence
    v[230, 1, 33] = special
    if what == "both":
        v[240, 1, 33] = float("inf")
        v[180, 0, 7], v[190, 0, 7] = float("inf"), float("-inf")
    _check(q, k, v, cu, label=what)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_keys_and_queries_that_are_no_numbers(dtype, dim):
    """A NaN key makes the rows that see it NaN, a NaN query its own row; the rest is as without them."""

    require_gpu()
    cu = [0, 150, 260]
    q, k, v = _inputs(16, 260, 260, 4, 2, dim, dtype)
    k[100, 1, 3] = float("nan")
    q[30, 0, 9] = float("nan")
    k[200, 0, 1] = float("inf")
    got = _op(q.cuda(), k.cuda(), v.cuda(), cu).cpu()
    nan = torch.zeros(260, 4, dtype=torch.bool)
    nan[100:150, 2:] = nan[30, 0] = True
    # an infinite key: scores of +inf make a row NaN, scores of -inf weigh nothing
    nan[200:, :2] = (q[200:, :2, 1] > 0)
    assert torch.equal(got.isnan().all(-1), nan) and torch.equal(got.isnan().any(-1), nan)
    clean_k, clean_q = k.clone(), q.clone()
    clean_k[100, 1, 3] = 0
    clean_q[30, 0, 9] = 0
    clean_k[200, 0, 1] = torch.finfo(dtype).max if dtype == F16 else 1e30
    want, bound = packed_attention64(clean_q, clean_k, v, cu, cu, dim ** -0.5)
    assert_within(got[~nan], want[~nan], bound[~nan])


def test_neighbours_are_not_read():
    """Rows before, between and behind the keys in use hold NaN."""

    require_gpu()
    lq, gaps = [40, 100, 7], [50, 130, 90]
    q, k, v = _inputs(17, sum(lq), sum(gaps), 8, 2, 128, BF16)
    cu_k, cu_q = offsets([40, 100, 7], start=20), offsets(lq)
    for x in (k, v):
        x[:20] = x[cu_k[-1]:] = float("nan")
    _check(q, k, v, cu_q, cu_k)


def test_offsets_out_of_order_leave_the_other_sequences_alone():
    require_gpu()
    q, k, v = _inputs(18, 200, 200, 4, 2, 128, BF16)
    cu = [0, 60, 40, 100, 5000]  # the second goes back, the fourth leaves the tensors
    got = _op(q.cuda(), k.cuda(), v.cuda(), cu, cu_k=cu).cpu()
    for a, b in ((0, 40), (60, 100)):
        first = 0 if a == 0 else 40
        want, bound = attention64(q[first:b], k[first:b], v[first:b], 128 ** -0.5)
        assert_within(got[a:b], want[a - first:], bound[a - first:], f"rows {a}..{b}")


def test_no_keys_and_no_queries():
    require_gpu()
    q, k, v = (x.cuda() for x in _inputs(22, 30, 30, 4, 2, 64, BF16))
    assert (_op(q, k[:0], v[:0], [0, 10, 30], cu_k=[0, 0, 0]) == 0).all()
    assert _op(q[:0], k, v, [0, 0], cu_k=[0, 30]).shape == (0, 4, 64)
    assert _op(q[:0], k[:0], v[:0], [0]).shape == (0, 4, 64)


def test_the_same_offsets_passed_twice_over_longer_keys():
    require_gpu()
    from prism_infer.ops.prompt_attention import prompt_attention

    q, k, v = _inputs(23, 50, 60, 4, 2, 128, BF16)
    cu = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu, num_heads=4, num_kv_heads=2, scale=0.1, cu_seqlens_k=cu)
    want, bound = packed_attention64(q, k, v, [0, 20, 50], [0, 20, 50], 0.1)
    assert_within(got, want, bound)


@pytest.mark.parametrize("batch", [40, 200, 3001])
def test_offsets_that_go_back_and_forth(batch):
    """Sequences that overlap write the same rows over and over, or not at all where they go back; nothing else."""

    require_gpu()
    q, k, v = (x.cuda() for x in _inputs(24, 150, 150, 2, 1, 64, BF16))
    cu = [150 * (i % 2) for i in range(batch + 1)]
    guard = torch.zeros(1 << 20, device="cuda")
    got = _op(q, k, v, cu)
    assert got.shape == q.shape and (guard == 0).all()
    want, bound = attention64(q.cpu(), k.cpu(), v.cpu(), 64 ** -0.5)
    assert_within(_op(q, k, v, [0, 150]), want, bound)


def test_captured_and_replayed_with_other_offsets_on_another_stream():
    require_gpu()
    from prism_infer.ops.prompt_attention import prompt_attention

    q, k, v = (x.cuda() for x in _inputs(19, 300, 300, 8, 2, 128, BF16))
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")

    def call():
        return prompt_attention(q, k, v, cu, num_heads=8, num_kv_heads=2, scale=0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for offs in ([0, 100, 300], [0, 17, 230], [0, 300, 300], [0, 100, 300]):
        cu.copy_(torch.tensor(offs, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, call()), offs
        torch.cuda.synchronize()
    assert torch.equal(out, eager)


def test_gradients_are_refused_where_recorded():
    require_gpu()
    q, k, v = (x.cuda() for x in _inputs(20, 8, 8, 2, 2, 64, BF16))
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        _op(q, k, v, [0, 8])
    with torch.no_grad():
        assert not _op(q, k, v, [0, 8]).requires_grad
