"""What the paged cache promises about calls that go wrong or sit out: tokens without a page, sessions without a new token,
the ends of the number range, reports across graph replays."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import paged_oracle
from tests.paged_helpers import Cache, check_attention, half_step
from world_engine_b200 import PagedSlab, ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def healthy():
    yield
    ops.check_status(torch.device("cuda"))


def reported():
    with pytest.raises(RuntimeError, match="page"):
        ops.check_status(torch.device("cuda"))


def queries(c, G, seed=1):
    g = torch.Generator().manual_seed(1000 + seed)
    return torch.randn(c.S, c.H * G, 1, c.Dh, generator=g).to(c.dtype).cuda()


def unname(c, *blocks):
    """Takes pages out of the table: (session, block, what stands there instead)."""
    for s, b, x in blocks:
        c.table_h[s, b] = x
    c.table.copy_(c.table_h)


# ------------------------------------------------------------------------------------------------ tokens without a page
@pytest.mark.parametrize("keep", [None, 96])
def test_a_dropped_token_is_not_held(keep):
    S, H, Dh, page = 3, 2, 64, 16
    slab = PagedSlab(S, H, Dh, BF16, page, 20, 96, **({} if keep is None else dict(keep=keep, sink=2, recent=8)))
    c = Cache(S, H, Dh, page, 6, BF16, lens=[0, 0, 0])
    c.kv, c.weights, c.positions = slab.kv, slab.weights, slab.positions
    c.table, c.lens, c.next_pos = slab.table, slab.lens, slab.next_pos
    slab.kv.fill_(float("nan"))                  # what a page holds before its tokens are written
    c.kv64, c.w64, c.pos64 = (x.cpu().numpy().copy() for x in (slab.kv.double(), slab.weights.double(), slab.positions))
    c.lens64, c.next64 = np.zeros((S, H), np.int32), np.zeros((S, H), np.int32)

    def step(T, seed):
        (k, v, _), (k64, v64, _) = c.new(T, seed=seed)
        slab.append(k, v)
        c.table64 = slab.table.cpu().numpy()
        if keep is None:
            paged_oracle.append(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64)
        else:
            paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, keep, 2, 8)
        c.assert_same_state()
        q = queries(c, 2, seed)
        before = c.w64.copy()
        out = slab.attend(q)
        check_attention(c, q, out, None, before, None if keep is None else slab.weights)
        c.w64 = slab.weights.double().cpu().numpy()
        return out

    slab.reserve(0, 20)                          # 32 slots
    slab.reserve(1, 16)
    out = step(40, 1)
    reported()
    assert c.lens64.tolist() == [[32, 32], [16, 16], [0, 0]] and torch.all(out[2] == 0)
    slab.reserve(0, 64)
    slab.reserve(2, 3)
    step(5, 2)
    reported()                                   # (session 1 has no more room)
    assert c.lens64.tolist() == [[37, 37], [16, 16], [5, 5]]
    slab.reserve(1, 17)
    step(1, 3)
    assert c.lens64.tolist() == [[38, 38], [17, 17], [6, 6]]


@pytest.mark.parametrize("T", [1, 7, 60, 900])
@pytest.mark.parametrize("budget", [None, (1000, 3, 40)])
@pytest.mark.parametrize("Dh,page,H", [(64, 16, 2), (128, 32, 1)])
def test_counts_stop_at_the_first_token_without_a_page(T, budget, Dh, page, H):
    lens = [0, page, 2 * page + 3, 5, page - 1, 10 * page, 3]
    c = Cache(len(lens), H, Dh, page, -(-1300 // page), BF16, seed=T, lens=lens)
    P = c.kv.shape[1]
    # missing: the first page, the next one, the one it is in the middle of, a later one, one far away, none, the table's bound
    unname(c, (0, 0, -1), (1, 1, P), (2, 2, -1), (3, 2, 2 ** 31 - 1), (4, 1, -1), (4, 2, -1), (6, 30, -2 ** 31))
    (k, v, w), (k64, v64, w64) = c.new(T, seed=5, with_weights=True)
    before = c.lens64.copy()
    if budget is None:
        ops.paged_append_(c.kv, c.table, c.lens, c.next_pos, k, v, None, c.weights, c.positions, w)
        paged_oracle.append(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, w64)
    else:
        ops.paged_append_evict_(c.kv, c.table, c.lens, c.next_pos, k, v, c.weights, c.positions, *budget, w_new=w)
        paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, *budget, w64)
    c.assert_same_state()
    reported()
    took = c.lens64 - before
    assert np.all(took[0] == 0) and np.all(took[1] == 0) and np.all(took[2] == 0) and np.all(took[5] == min(T, 1000 - 10 * page if budget else T))
    assert np.all(took[3] == min(T, 2 * page - 5)) and np.all(took[4] == 1)


def test_a_long_append_stops_where_its_pages_do():
    # more pages than one look of the CTA at the table; clusters of CTAs
    for at in (0, 31, 32, 257, 1200):
        c = Cache(1, 1, 64, 16, 1250, F16, seed=at, lens=[9])
        unname(c, (0, at, -1), (0, at + 7, -1))
        (k, v, _), (k64, v64, _) = c.new(19900, seed=6)
        ops.paged_append_(c.kv, c.table, c.lens, c.next_pos, k, v, weights=c.weights, positions=c.positions)
        paged_oracle.append(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64)
        c.assert_same_state()
        reported()
        assert int(c.lens64[0, 0]) == max(16 * at, 9)


# ------------------------------------------------------------------------------------------------ held slots without a page
@pytest.mark.parametrize("lens,T,keep,sink,recent,blocks", [
    ([64, 64], 3, 64, 2, 20, [(0, 1)]),                  # at the budget
    ([64, 60], 1, 64, 2, 62, [(0, 0), (1, 2)]),          # all the rest is shielded: the newest of them go without a slot
    ([90, 70], 3, 50, 1, 30, [(0, 1), (0, 4), (1, 3)]),  # the budget was lowered: slots of either side
    ([90, 70], 0, 20, 0, 0, [(0, 2), (0, 3), (0, 4), (0, 5), (1, 0)]),
    ([48, 64], 200, 64, 4, 16, [(0, 0), (1, 3)]),        # a prompt
    ([64, 48], 79, 64, 4, 30, [(0, 0), (0, 2), (0, 3), (1, 0), (1, 1)]),   # ... fewer slots than shielded tokens
    ([64, 64], 5, 64, 0, 0, [(0, 0), (0, 1), (0, 2), (0, 3)])])   # no page at all
@pytest.mark.parametrize("with_weights", [False, True])
def test_eviction_neither_keeps_nor_fills_a_slot_without_a_page(lens, T, keep, sink, recent, blocks, with_weights):
    c = Cache(2, 2, 64, 16, 6, BF16, seed=T + keep, lens=lens)
    for s in range(2):                                   # odd weights among them: the last word must not be theirs
        c.weights[c.table[s, 0].long(), 0, 3] = float("inf")
        c.weights[c.table[s, 0].long(), 0, 5] = float("nan")
        c.weights[c.table[s, 0].long(), 1, 3] = float("-inf")
    c.w64 = c.weights.double().cpu().numpy()
    unname(c, *((s, b, -1) for s, b in blocks))
    (k, v, w), (k64, v64, w64) = c.new(T, seed=7, with_weights=with_weights)
    ops.paged_append_evict_(c.kv, c.table, c.lens, c.next_pos, k, v, c.weights, c.positions, keep, sink, recent, w_new=w)
    paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, keep, sink, recent, w64)
    c.assert_same_state()
    reported()


@pytest.mark.parametrize("H,idle,held,keep,T", [(1, 0, 20000, 20000, 50), (3, 120, 5400, 5300, 9), (2, 0, 40000, 33333, 17)])
def test_long_evictions_around_slots_without_a_page(H, idle, held, keep, T):
    # clusters; CTAs that go through their candidates in rounds (beside sessions that hold nothing)
    c = Cache(2, H, 64, 64, -(-held // 64), F16, seed=H, lens=[held, held - 1])
    unname(c, (0, 0, -1), (0, 50, -1), (0, held // 64 - 1, c.kv.shape[1]), (1, keep // 64, -1))
    (k, v, w), (k64, v64, w64) = c.new(T, seed=8, with_weights=True)

    def padded(x, value=0):
        return torch.cat([x, torch.full((idle, *x.shape[1:]), value, dtype=x.dtype, device="cuda")])
    table, lens, next_pos = padded(c.table, -1), padded(c.lens), padded(c.next_pos)
    n_new = torch.tensor([T, T] + [0] * idle, dtype=torch.int32, device="cuda")
    ops.paged_append_evict_(c.kv, table, lens, next_pos, padded(k), padded(v), c.weights, c.positions, keep, 4, 100, n_new, padded(w))
    assert not lens[2:].any() and not next_pos[2:].any()
    c.lens, c.next_pos = lens[:2], next_pos[:2]
    paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, keep, 4, 100, w64)
    c.assert_same_state()
    reported()


# ------------------------------------------------------------------------------------------------ sessions that sit out
@pytest.mark.parametrize("S,H,G,page,M,most", [
    (6, 2, 1, 16, 8, 128),            # never split
    (6, 2, 4, 16, 40, 640),           # split and joined
    (14, 5, 20, 16, 512, 8192),       # runs handed out, two units per kv head
    (140, 3, 2, 32, 6, 190)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_a_session_that_sits_out_is_left_alone(S, H, G, page, M, most, accumulate):
    lens = [[(most * (1 + (7 * s + 3 * h) % 11)) // 11 if most < 1000 else most - 13 * s - h for h in range(H)] for s in range(S)]
    c = Cache(S, H, 64, page, M, BF16, seed=S, lens=lens)
    q = queries(c, G)
    out_of_step = [s for s in range(S) if s % 3 == 1]
    q[out_of_step] = float("nan")                        # rows of a padded batch
    n_new = torch.ones(S, dtype=torch.int32, device="cuda")
    n_new[out_of_step] = 0
    n_new[out_of_step[-1]] = -1
    n_new[0] = 7
    weights = c.weights if accumulate else None
    lse = torch.zeros(S, H * G, device="cuda")
    out = ops.paged_attn(q, c.kv, c.table, c.lens, weights=weights, lse=lse, n_new=n_new)
    assert torch.all(out[out_of_step] == 0) and torch.all(torch.isneginf(lse[out_of_step]))
    before = c.w64.copy()
    c.lens64[out_of_step] = 0                            # as if they held nothing
    check_attention(c, torch.where(n_new[:, None, None, None] > 0, q, 0.0), out, lse, before, weights)
    if accumulate:
        pages = c.table[out_of_step].long().flatten()
        assert torch.equal(c.weights[pages].double().cpu().nan_to_num(7.0), torch.from_numpy(before)[pages.cpu()].nan_to_num(7.0))
    held = c.lens.clone()
    held[out_of_step] = 0
    c.weights.copy_(torch.from_numpy(before).float())
    assert torch.equal(out, ops.paged_attn(q, c.kv, c.table, held, weights=weights))


@pytest.mark.parametrize("budget", [dict(), dict(keep=20, sink=1, recent=4)])
@pytest.mark.parametrize("compiled", [False, True])
def test_a_step_that_some_sessions_sit_out(budget, compiled):
    """A padded step leaves the sessions that sit out as they were, and the others as steps without them do."""
    def slab():
        x = PagedSlab(3, 2, 64, BF16, 16, 12, 48, **budget)
        for s in range(3):
            x.reserve(s, 20 if budget else 48)
        return x
    every, alone = slab(), [PagedSlab(1, 2, 64, BF16, 16, 4, 48, **budget) for _ in range(3)]
    for x in alone:
        x.reserve(0, 20 if budget else 48)
    g = torch.Generator().manual_seed(2)
    step = every.append_and_attend
    if compiled:
        step = torch.compile(lambda q, k, v, n: every.append_and_attend(q, k, v, n), fullgraph=True, backend="aot_eager")
    for i in range(30):
        q, k, v = (torch.randn(3, n, 1, 64, generator=g).to(BF16).cuda() for n in (4, 2, 2))
        n_new = torch.tensor([1, i % 2, i % 3 != 0], dtype=torch.int32)
        idle = [s for s in range(3) if n_new[s] == 0]
        for x in (q, k, v):
            x[idle] = float("nan")
        with torch.no_grad():
            y = step(q, k, v, n_new.cuda())
        for s in range(3):
            if s in idle:
                assert torch.all(y[s] == 0)
            else:
                z = alone[s].append_and_attend(q[s:s + 1], k[s:s + 1], v[s:s + 1]).float()
                # (cut into other runs, so sums are added up in another order: two roundings to bf16 and 2^-13 of the
                # largest values in between, where weights are held to 2^-16)
                assert torch.allclose(y[s].float(), z[0], rtol=2 ** -7, atol=2 ** -11)
    for s in range(3):
        assert torch.equal(every.lens[s], alone[s].lens[0]) and torch.equal(every.next_pos[s], alone[s].next_pos[0])
        assert torch.isfinite(every.weights).all()
    assert every.next_pos[:, 0].tolist() == [30, 15, 20]


def test_traces_with_permuted_queries():
    c = Cache(3, 2, 64, 16, 9, BF16, seed=4, lens=[100, 3, 144])
    x = torch.randn(8, 3, 1, 64, device="cuda").to(BF16)

    def step(x):
        y = ops.paged_attn_op(x.transpose(0, 1), c.kv, c.table, c.lens, 0.0, None)
        return y.transpose(0, 1).reshape(8, -1) + 1, y
    with torch.no_grad():
        flat, y = torch.compile(step, fullgraph=True, backend="aot_eager")(x)
        want_flat, want = step(x)
    assert torch.equal(y, want) and y.stride() == want.stride() and torch.equal(flat, want_flat)
    q = x.transpose(0, 1)
    check_attention(c, q, y)


def test_a_captured_step_whose_sessions_come_and_go():
    def slab():
        x = PagedSlab(4, 2, 128, BF16, 16, 16, 64, keep=40, sink=1, recent=4)
        for s in range(4):
            x.reserve(s, 40)
        return x
    eager, graphed = slab(), slab()
    g = torch.Generator().manual_seed(8)
    steps = [[torch.randn(4, n, 1, 128, generator=g).to(BF16).cuda() for n in (4, 2, 2)] +
             [torch.randint(0, 2, (4,), generator=g, dtype=torch.int32).cuda()] for _ in range(60)]
    held = [x.clone() for x in steps[0]]
    held[3].zero_()
    graphed.append_and_attend(*held)                     # (everybody sits out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = graphed.append_and_attend(*held)
    for i, step in enumerate(steps):
        want = eager.append_and_attend(*step)
        for a, b in zip(held, step):
            a.copy_(b)
        graph.replay()
        assert torch.equal(y, want), i
        assert torch.all(y[step[3] == 0] == 0)
    for name in ("kv", "weights", "positions", "lens", "next_pos"):
        assert torch.equal(getattr(eager, name), getattr(graphed, name)), name


# ------------------------------------------------------------------------------------------------ numbers
def one_column(c, logits, scale=1.0):
    """Keys whose only column is the logit (times 1/scale): the logits of q = 1 in that column are exact."""
    n = len(logits)
    i = torch.arange(n)
    pg, row = c.table_h[0, i // c.page].long(), i % c.page
    k = torch.zeros(n, c.Dh, dtype=c.dtype)
    k[:, 0] = logits.to(c.dtype)
    c.kv[0, pg.cuda(), 0, row.cuda()] = k.cuda()
    c.kv64[0, pg, 0, row] = k.double().numpy()
    return pg, row, k[:, 0].double()


def put_values(c, pg, row, v):
    c.kv[1, pg.cuda(), 0, row.cuda()] = v.cuda()
    c.kv64[1, pg, 0, row] = v.double().numpy()


def ones_in_column_0(c, G=1, x=1.0):
    q = torch.zeros(1, G, 1, c.Dh, dtype=c.dtype, device="cuda")
    q[..., 0] = x
    return q


def narrowed(x, dtype):
    return x.to(dtype).double()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n", [300, 1500])
def test_weights_are_held_in_more_than_16_bits(dtype, n):
    """Values chosen against the rounding of the weights: each has the sign of what rounding its weight to 16 bits would
    lose, and half of them cancel the other half.  Logits lie in one column, so they are exact but for the scaling: with
    |x| <= 6, x log2 e is off by 6 * 1.5 * 2^-23 < 2^-19 and e^x by 2^-19 of itself, 2^x of the GPU by 2^-21, twice for
    the normalisation (2^-17 in all).  A weight as the sum of two 16-bit numbers is off by half a step of half a step.
    Sums are held in fp32, 16 products to an addition that may truncate, in runs joined in fp32: at most n / 16 + 64
    steps of 2^-23."""
    c = Cache(1, 1, 64, 16, -(-n // 16), dtype, seed=3, lens=[n])
    g = torch.Generator().manual_seed(n)
    logits = -6 * torch.rand(n, generator=g)
    logits[::64] = 0.0                                   # the reference of every tile
    pg, row, x = one_column(c, logits)
    e = torch.exp(x)
    lost = e - narrowed(e, dtype)
    v = torch.where(lost >= 0, 1.0, -1.0)[:, None].expand(n, 64).to(dtype).contiguous()
    put_values(c, pg, row, v)
    p = e / e.sum()
    want, spread = float((p * v[:, 0].double()).sum()), 1.0
    u = half_step(dtype)
    tol = (2.0 ** -17 + u * u + (n / 16 + 64) * 2.0 ** -23) * spread + u * abs(want)
    single = float((narrowed(e, dtype) * v[:, 0].double()).sum() / e.sum())
    assert abs(single - want) > 1.5 * tol                # what the tolerance is there to see
    got = ops.paged_attn(ones_in_column_0(c), c.kv, c.table, c.lens, scale=1.0).double()
    assert float((got - want).abs().max()) <= tol


@pytest.mark.parametrize("G", [1, 3, 16])
@pytest.mark.parametrize("n,drop", [(100000, 25.6), (100000, 31.0), (2000, 24.3)])
def test_many_small_weights_count_in_fp16(G, n, drop):
    """One token takes nearly all of the weight and its value is 0; all others have weights that 16 bits cannot hold on
    their own, and value 1: the output is what they have in all.  The logits are exact (multiples of 2^-4 below 32); their
    log2 e multiple is off by 2 * 2^-24 * 45 < 2^-17 (natural: the weights by that), sums as above."""
    c = Cache(1, 1, 64, 32, -(-n // 32), F16, seed=4, lens=[n])
    x0 = round(drop * np.log(2) * 16) / 16
    for first in (0, n - 1, n // 2):
        logits = torch.full((n,), -x0)
        logits[first] = 0.0
        pg, row, x = one_column(c, logits)
        v = torch.ones(n, 64, dtype=F16)
        v[first] = 0.0
        put_values(c, pg, row, v)
        p = torch.exp(x)
        p /= p.sum()
        want = float(p.sum() - p[first])
        got = ops.paged_attn(ones_in_column_0(c, G), c.kv, c.table, c.lens, scale=1.0).double()
        tol = want * (half_step(F16) + 2.0 ** -15 + (n / 16 + 64) * 2.0 ** -23) + 2.0 ** -25
        assert float((got - want).abs().max()) <= tol

def test_logits_at_the_far_end_of_the_range():
    # logits of -1.5e38 to -2e38: the softmax goes by their differences all the same
    n = 300
    c = Cache(1, 1, 64, 16, 20, BF16, seed=5, lens=[n])
    logits = -torch.linspace(1.5e19, 2e19, n)
    pg, row, _ = one_column(c, logits)
    out = ops.paged_attn(ones_in_column_0(c, 1, 1e19), c.kv, c.table, c.lens, scale=1.0)
    top = (c.kv64[0, pg, 0, row][:, 0] == c.kv64[0, pg, 0, row][:, 0].max())
    want = c.kv64[1, pg, 0, row][top].mean(axis=0)       # of equal ones the mean
    spread = np.abs(c.kv64[1, pg, 0, row][top]).mean(axis=0)
    got = out[0, 0, 0].double().cpu().numpy()
    assert np.all(np.abs(got - want) <= half_step(BF16) * np.abs(want) + 2.0 ** -15 * spread)

# ------------------------------------------------------------------------------------------------ reports
CHILD = """
import torch
from world_engine_b200 import PagedSlab, ops
slab = PagedSlab(1, 2, 64, torch.bfloat16, 16, 4, 32)
slab.reserve(0, 32)
x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):                 # the first calls of the process
    slab.append_and_attend(x, x, x)
dev = torch.device("cuda")
ops.check_status(dev)
page = int(slab.table[0, 0])
slab.table[0, 0] = -1
graph.replay()
slab.table[0, 0] = page
graph.replay()
try:
    ops.check_status(dev)
except RuntimeError as e:
    print("reported", e)
ops.check_status(dev)
"""


def test_a_report_outlives_the_next_replay():
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert "reported" in r.stdout and "page" in r.stdout


# ------------------------------------------------------------------------------------------------ arguments that steps rarely give
@pytest.mark.parametrize("lens,T", [([40, 50], 6), ([10, 0], 6), ([50, 50], 0)])
def test_eviction_into_other_counts(lens, T):
    c = Cache(2, 3, 64, 16, 4, BF16, seed=T, lens=lens)
    (k, v, w), (k64, v64, w64) = c.new(T, seed=3, with_weights=True)
    held, given = c.lens.clone(), c.next_pos.clone()
    lens_out, next_pos_out = torch.full_like(held, -7), torch.full_like(held, -7)
    ops.paged_append_evict_(c.kv, c.table, c.lens, c.next_pos, k, v, c.weights, c.positions, 44, 2, 9, w_new=w, lens_out=lens_out,
                            next_pos_out=next_pos_out)
    assert torch.equal(c.lens, held) and torch.equal(c.next_pos, given)
    paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, 44, 2, 9, w64)
    c.lens, c.next_pos = lens_out, next_pos_out
    c.assert_same_state()


def test_a_prompt_with_weights_into_a_budgeted_slab():
    # w_new as a view with strides of its own, a padded batch
    S, H, Dh, page, keep, T = 3, 2, 128, 16, 30, 100
    slab = PagedSlab(S, H, Dh, F16, page, 8, 4096, keep=keep, sink=2, recent=6)
    for s in range(S):
        slab.reserve(s, 4096)
    c = Cache(S, H, Dh, page, 2, F16, lens=[0] * S)
    (k, v, w), (k64, v64, w64) = c.new(T, seed=4, with_weights=True)
    n_new = torch.tensor([100, 17, 31], dtype=torch.int32)
    kv64, w_64, pos64 = (x.cpu().numpy().copy() for x in (slab.kv.double(), slab.weights.double(), slab.positions))
    lens64, next64 = np.zeros((S, H), np.int32), np.zeros((S, H), np.int32)
    slab.append(k, v, n_new.cuda(), w.transpose(0, 2).contiguous().transpose(0, 2))
    paged_oracle.append_evict(kv64, slab.table.cpu().numpy(), lens64, next64, k64, v64, n_new, w_64, pos64, keep, 2, 6, w64)
    assert np.array_equal(slab.kv.double().cpu().numpy(), kv64) and np.array_equal(slab.weights.double().cpu().numpy(), w_64)
    assert np.array_equal(slab.positions.cpu().numpy(), pos64) and np.array_equal(slab.lens.cpu().numpy(), lens64)
    assert lens64.tolist() == [[30, 30], [17, 17], [30, 30]]
