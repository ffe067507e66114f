"""GPU step metadata against a plain loop, every value equal."""

from __future__ import annotations

import pytest
import torch

from _helpers import require_gpu

pytestmark = pytest.mark.gpu

FITS = 2**31 - 1


def plain(tables, cached, new, page, rows, free, start=0):
    """The definition, request by request; a request's blocks past the table or the free list are missing (-1)."""

    width, used, misfit = tables.shape[1], max(start, 0), FITS
    slots, positions, cu, out = [-1] * rows, [0] * rows, [0], []
    for i, (row, c, n) in enumerate(zip(tables.tolist(), cached, new)):
        bad = c < 0 or n < 0 or start < 0 or max(c, 0) + max(n, 0) > width * page
        c, n = max(c, 0), max(n, 0)
        held, need = min(-(-c // page), width), min(-(-(c + n) // page), width)
        blocks = row[:held] + [free[e] if e < len(free) else -1 for e in range(used, used + need - held)]
        used += need - held
        for j in range(min(n, max(rows - cu[-1], 0))):
            p, t = c + j, cu[-1] + j
            positions[t] = p
            if p // page < width and blocks[p // page] >= 0:
                slots[t] = blocks[p // page] * page + p % page
        cu.append(cu[-1] + n)
        if bad or cu[-1] > rows or used > len(free):
            misfit = min(misfit, i)
        out.append(blocks + [-1] * (width - len(blocks)))
    ctx = [max(c, 0) + max(n, 0) for c, n in zip(cached, new)]
    return dict(slot_mapping=slots, positions=positions, cu_seqlens_q=cu, context_lens=ctx, max_context_len=max(ctx, default=0),
                next_free=used, first_misfit=misfit, block_tables=out)


def _cuda(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _build(tables, cached, new, page, rows, free, **kw):
    from prism_infer.engine.step_metadata import build_step_metadata

    return build_step_metadata(tables.cuda(), _cuda(cached), _cuda(new), block_size=page, num_tokens=rows,
                               free_blocks=_cuda(free), **kw)


def _same(m, want):
    for name, value in want.items():
        assert getattr(m, name).tolist() == value, name


def _case(seed, batch, page, most_cached, most_new, *, spare_width=2, pad=0):
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(0, most_cached + 1, (batch,), generator=g).tolist()
    new = torch.randint(0, most_new + 1, (batch,), generator=g).tolist()
    width = -(-(most_cached + most_new) // page) + spare_width
    held = [-(-c // page) for c in cached]
    need = [-(-(c + n) // page) for c, n in zip(cached, new)]
    perm = torch.randperm(sum(need) + 5, generator=g).to(torch.int32)
    tables = torch.randint(-5, 10**6, (batch, width), generator=g, dtype=torch.int32)
    at = 0
    for i, n in enumerate(held):
        tables[i, :n] = perm[at:at + n]
        at += n
    return tables, cached, new, page, sum(new) + pad, perm[at:].tolist()


@pytest.mark.parametrize("batch,page,most_cached,most_new,pad", [
    (1, 256, 0, 1, 0), (1, 16, 5000, 3000, 0), (3, 16, 40, 17, 5), (64, 256, 16000, 1, 0), (32, 64, 900, 500, 333),
    (255, 16, 64, 3, 0), (256, 16, 64, 3, 1), (257, 48, 64, 3, 2), (1000, 1, 9, 9, 0), (1024, 16, 300, 40, 63),
    (5, 100, 0, 1000, 0), (8192, 16, 20, 2, 3), (40, 16, 100, 0, 7)])
def test_against_the_definition(batch, page, most_cached, most_new, pad):
    require_gpu()
    case = _case(batch + page, batch, page, most_cached, most_new, pad=pad)
    m = _build(*case)
    _same(m, plain(*case))
    m.check()


def test_no_requests_and_no_tokens():
    require_gpu()
    _same(_build(torch.zeros(0, 4, dtype=torch.int32), [], [], 16, 6, []), plain(torch.zeros(0, 4), [], [], 16, 6, []))
    case = (torch.tensor([[7, -1]], dtype=torch.int32), [16], [0], 16, 0, [])
    _same(_build(*case), plain(*case))
    case = (torch.zeros(3, 0, dtype=torch.int32), [0, 0, 5], [0, 2, 1], 16, 8, [4])  # tables without entries
    _same(_build(*case), plain(*case))


@pytest.mark.parametrize("what", ["free", "width", "tokens", "negative", "start", "held", "huge"])
def test_requests_that_do_not_fit(what):
    require_gpu()
    tables, cached, new, page, rows, free = _case(1, 20, 16, 90, 40)
    start = 0
    if what == "free":
        free = free[:len(free) // 2]
    elif what == "width":
        tables = tables[:, :5].contiguous()
    elif what == "tokens":
        rows //= 3
    elif what == "negative":
        cached[4], new[9] = -3, -70000
    elif what == "start":
        start = -2
    elif what == "held":
        new[3], cached[3] = 5, 20
        tables[3, 1] = -1  # a held block that is none: its tokens have no slot (and the lengths no longer fit the rows)
    else:
        cached[7], new[8] = FITS, FITS
    m = _build(tables, cached, new, page, rows, free, free_start=_cuda([start]))
    want = plain(tables, cached, new, page, rows, free, start)
    if what == "huge":  # offsets, lengths and positions stay at INT32_MAX
        want["positions"] = [min(x, FITS) for x in want["positions"]]
        want["cu_seqlens_q"] = [min(x, FITS) for x in want["cu_seqlens_q"]]
        want["context_lens"] = [min(x, FITS) for x in want["context_lens"]]
        want["max_context_len"] = FITS
    _same(m, want)
    assert want["first_misfit"] != FITS
    with pytest.raises(RuntimeError, match=f"request {want['first_misfit']} does not fit"):
        m.check()


def test_slots_past_int32_are_missing():
    require_gpu()
    page = 256
    tables = torch.tensor([[2**23 - 1, 2**23]], dtype=torch.int32)
    m = _build(tables, [page], [page], page, page, [2**23])
    assert m.slot_mapping.tolist() == [-1] * page
    m = _build(tables, [page - 2], [2], page, 2, [])
    assert m.slot_mapping.tolist() == [2**31 - 2, 2**31 - 1]


def test_strided_tables_and_steps_in_a_row():
    """A prompt step, then decode steps, each from the one before, without a host copy; buffers filled in place."""

    require_gpu()
    from prism_infer.engine.step_metadata import build_step_metadata

    page, batch, width = 16, 9, 12
    g = torch.Generator().manual_seed(2)
    free = torch.randperm(120, generator=g).to(torch.int32)
    wide = torch.full((width, 2 * batch), -9, dtype=torch.int32, device="cuda").t()[::2]
    zeros = torch.zeros(batch, dtype=torch.int32, device="cuda")
    new = torch.randint(1, 60, (batch,), generator=g, dtype=torch.int32)
    m = build_step_metadata(wide, zeros, new.cuda(), block_size=page, num_tokens=int(new.sum()), free_blocks=free.cuda())
    tables, cached, start = torch.full((batch, width), -9), [0] * batch, 0
    want = plain(tables, cached, new.tolist(), page, int(new.sum()), free.tolist())
    _same(m, want)
    buffers = [None, None]
    one = torch.ones(batch, dtype=torch.int32, device="cuda")
    for step in range(40):
        at = step % 2
        m = build_step_metadata(m.block_tables, m.context_lens, one, block_size=page, num_tokens=batch,
                                free_blocks=free.cuda(), free_start=m.next_free, out=buffers[at])
        buffers[at] = m
        want = plain(torch.tensor(want["block_tables"]), want["context_lens"], [1] * batch, page, batch, free.tolist(),
                     want["next_free"])
        _same(m, want)
    m.check()
    with pytest.raises(ValueError, match="shares memory"):
        build_step_metadata(m.block_tables, m.context_lens, one, block_size=page, num_tokens=batch, out=m)
    with pytest.raises(ValueError, match="other sizes"):
        build_step_metadata(buffers[0].block_tables, buffers[0].context_lens, one, block_size=page, num_tokens=batch + 4, out=m)


def test_captured_with_lengths_of_the_replay():
    require_gpu()
    from prism_infer.engine.step_metadata import build_step_metadata

    tables, cached, new, page, rows, free = _case(3, 30, 16, 200, 20, pad=100)
    t, c, n, f = tables.cuda(), _cuda(cached), _cuda(new), _cuda(free)

    def call():
        return build_step_metadata(t, c, n, block_size=page, num_tokens=rows, free_blocks=f)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m = call()
    for k in (0, 1, 2):
        lens = [max(x - k, 0) for x in new]
        n.copy_(_cuda(lens))
        graph.replay()
        _same(m, plain(tables, cached, lens, page, rows, free))
