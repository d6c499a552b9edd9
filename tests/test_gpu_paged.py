"""The paged cache's operators on the GPU against their 64-bit restatement: lengths from nothing to long ones, pages that
end inside a tile, shared heads, strides, padded batches, budgets, streams and graphs."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle
from tests.paged_helpers import Cache, check_attention
from world_engine_b200 import PagedSlab, ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def healthy():
    yield
    ops.check_status(torch.device("cuda"))


def queries(c, G, seed=1, gain=1.0):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(c.S, c.H * G, 1, c.Dh, generator=g) * gain).to(c.dtype).cuda()


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_at_every_page_size(Dh, page, dtype):
    lens = [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 300]
    c = Cache(len(lens), 2, Dh, page, -(-320 // page), dtype, seed=page + Dh, lens=lens)
    q = queries(c, 2)
    lse = torch.empty(c.S, 4, device="cuda")
    out = ops.paged_attn(q, c.kv, c.table, c.lens, lse=lse)
    check_attention(c, q, out, lse)
    assert torch.all(out[0] == 0) and torch.all(torch.isneginf(lse[0]))


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 12, 16, 17, 33, 64])
@pytest.mark.parametrize("Dh", [64, 128])
def test_attention_with_shared_heads(G, Dh):
    c = Cache(3, 2, Dh, 32, 20, BF16, seed=G, lens=[513, 40, 1])
    q = queries(c, G)
    before = c.w64.copy()
    out = ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights)
    check_attention(c, q, out, None, before, c.weights)


@pytest.mark.parametrize("S,H,G,lens", [
    (1, 1, 1, [9000]), (1, 3, 2, [20011]), (2, 1, 8, [12345, 3]), (40, 5, 1, None), (1, 16, 1, [4096]), (7, 16, 4, None)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_attention_of_long_and_ragged_batches(S, H, G, lens, accumulate):
    if lens is None:
        lens = [[(s * 379 + h * 97) % 1500 for h in range(H)] for s in range(S)]        # heads hold different numbers
    c = Cache(S, H, 128, 64, -(-int(np.max(lens)) // 64) + 1, BF16, seed=S, lens=lens)
    q = queries(c, G)
    before = c.w64.copy()
    lse = torch.empty(S, H * G, device="cuda")
    out = ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights if accumulate else None, lse=lse)
    check_attention(c, q, out, lse, before, c.weights if accumulate else None)


@pytest.mark.parametrize("S,H,G,page,lens", [
    (5, 16, 1, 64, [8192, 8000, 8191, 7777, 8100]),          # long runs: their ends are handed out one by one
    (9, 5, 20, 16, [8192, 6000, 0, 8191, 7001, 1, 8180, 8100, 7900]),   # ... with two units per kv head
    (2, 3, 4, 32, [120001, 119000])])
def test_attention_where_runs_are_handed_out(S, H, G, page, lens):
    c = Cache(S, H, 64, page, -(-max(lens) // page), BF16, seed=S, lens=lens)
    q = queries(c, G)
    before = c.w64.copy()
    out = ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights)
    check_attention(c, q, out, None, before, c.weights)
    first = c.weights.clone()
    for _ in range(3):                                       # whoever takes a run, the result is the same
        c.weights.copy_(torch.from_numpy(c.w64).float())
        assert torch.equal(ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights), out)
        assert torch.equal(c.weights.nan_to_num(), first.nan_to_num())


@pytest.mark.parametrize("G", [1, 3, 16, 20])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_attention_of_sessions_that_are_never_split(G, page):
    lens = [[(s * 31 + h * 47) % 129 for h in range(3)] for s in range(70)]      # more heads than SMs, some hold nothing
    c = Cache(70, 3, 128, page, 128 // page, F16, seed=G, lens=lens)
    q = queries(c, G)
    lse = torch.empty(70, 3 * G, device="cuda")
    check_attention(c, q, ops.paged_attn(q, c.kv, c.table, c.lens, lse=lse), lse)


def test_pages_beyond_32_bits_of_elements():
    # offsets of more than 2^31 elements within a plane of the pool, and K and V planes as far apart
    H, page, Dh = 2, 256, 128
    P = (1 << 31) // (H * page * Dh) + 40
    kv = torch.empty(2, P, H, page, Dh, dtype=BF16, device="cuda")
    weights, positions = torch.zeros(P, H, page, device="cuda"), torch.zeros(P, H, page, dtype=torch.int32, device="cuda")
    table = torch.tensor([[P - 1, 3, P - 20, P - 7]], dtype=torch.int32, device="cuda")
    small = Cache(1, H, Dh, page, 4, BF16, seed=2, lens=[0])
    for far, near in ((kv, small.kv), (weights, small.weights), (positions, small.positions)):
        if far is kv:
            far[:, table[0].long()] = near[:, small.table[0].long()]
        else:
            far[table[0].long()] = near[small.table[0].long()]
    lens, next_pos = small.lens.clone(), small.next_pos.clone()
    for T, keep in ((700, 1000), (600, 1000)):
        (k, v, w), _ = small.new(T, seed=T, with_weights=True)
        ops.paged_append_evict_(kv, table, lens, next_pos, k, v, weights, positions, keep, 4, 100, w_new=w)
        ops.paged_append_evict_(small.kv, small.table, small.lens, small.next_pos, k, v, small.weights, small.positions, keep,
                                4, 100, w_new=w)
    q = queries(small, 2)
    out = ops.paged_attn(q, kv, table, lens, weights=weights)
    assert torch.equal(out, ops.paged_attn(q, small.kv, small.table, small.lens, weights=small.weights))
    t, u = table[0].long(), small.table[0].long()
    assert torch.equal(kv[:, t].view(torch.int16), small.kv[:, u].view(torch.int16))
    assert torch.equal(weights[t].nan_to_num(), small.weights[u].nan_to_num()) and torch.equal(positions[t], small.positions[u])
    (k, v, _), _ = small.new(3, seed=9)
    ops.paged_append_(kv, table, lens, next_pos, k, v)
    assert torch.equal(kv[0, P - 7, :, 1000 - 768:1003 - 768], k[0].contiguous())


@pytest.mark.parametrize("S,H", [(13, 32), (25, 16), (96, 4), (385, 1), (103, 8), (416, 2), (417, 3), (5, 250)])
def test_attention_at_every_share_of_the_set_up(S, H):
    # as many heads as the set-up has threads, a few less, more, and multiples of them
    lens = [[(s * 37 + h * 11) % 150 for h in range(H)] for s in range(S)]
    c = Cache(S, H, 64, 16, 10, BF16, seed=S, lens=lens)
    q = queries(c, 1)
    before = c.w64.copy()
    lse = torch.empty(S, H, device="cuda")
    check_attention(c, q, ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights, lse=lse), lse, before, c.weights)


@pytest.mark.parametrize("gain", [0.0, 8.0, 40.0])
def test_attention_with_flat_and_peaked_softmax(gain):
    # gain 40: logits of some hundreds, the running maximum rises many times; 0: all weights equal
    c = Cache(2, 2, 128, 16, 70, BF16, seed=5, lens=[1100, 1111])
    q = queries(c, 4, gain=gain)
    before = c.w64.copy()
    out = ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights)
    check_attention(c, q, out, None, before, c.weights)


def test_attention_when_logits_rise_with_every_token():
    c = Cache(1, 1, 64, 16, 130, F16, seed=6, lens=[2048])
    ramp = torch.linspace(-30, 30, 2048)
    i = torch.arange(2048)
    pg, row = c.table_h[0, i // 16].long(), i % 16
    k = torch.zeros(2048, 64, dtype=F16)
    k[:, 0] = ramp
    c.kv[0, pg.cuda(), 0, row.cuda()] = k.cuda()
    c.kv64[0, pg, 0, row] = k.double().numpy()
    q = torch.zeros(1, 1, 1, 64, dtype=F16, device="cuda")
    q[..., 0] = 8.0
    out = ops.paged_attn(q, c.kv, c.table, c.lens)
    check_attention(c, q, out)


def test_attention_takes_strided_tensors_and_a_scale():
    c = Cache(3, 2, 128, 32, 9, BF16, seed=7, lens=[257, 31, 100], nhd=True)
    wide = torch.randn(3, 1, 3, 6, 128, device="cuda").to(BF16)
    q = wide[:, :, 1].transpose(1, 2)                                   # [S, Hq, 1, Dh] out of a merged projection
    hold = torch.full((3, 1, 6, 256), 7.0, dtype=BF16, device="cuda")
    out = hold[..., :128].transpose(1, 2)
    got = ops.paged_attn(q, c.kv, c.table, c.lens, scale=0.25, out=out)
    assert got is out
    check_attention(c, q, out, scale=0.25)
    assert torch.all(hold[..., 128:] == 7.0)
    table = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")   # a table wider than the sessions need
    table[:, :9] = c.table
    assert torch.equal(ops.paged_attn(q, c.kv, table[:, :9], c.lens, scale=0.25), out)
    assert torch.equal(ops.paged_attn(q, c.kv, table, c.lens, scale=0.25), out)


def test_attention_over_other_orders_of_the_pool():
    # K and V of a page next to each other, pages last, heads first: any strides will do
    c = Cache(3, 2, 64, 16, 30, F16, seed=17, lens=[450, 31, 480])
    q = queries(c, 4)
    want = ops.paged_attn(q, c.kv, c.table, c.lens)
    for order in ((1, 0, 2, 3, 4), (2, 1, 0, 3, 4), (3, 1, 2, 0, 4), (2, 3, 0, 1, 4)):
        back = [order.index(i) for i in range(5)]
        kv = c.kv.permute(order).contiguous().permute(back)
        assert kv.shape == c.kv.shape and torch.equal(ops.paged_attn(q, kv, c.table, c.lens), want)
    with pytest.raises(ValueError, match="out must not"):
        ops.paged_attn(q, c.kv, c.table, c.lens, out=q)


@pytest.mark.parametrize("page,M", [(16, 8), (16, 40)])
def test_attention_when_nobody_holds_anything(page, M):
    c = Cache(3, 2, 128, page, M, BF16, seed=18, lens=[0, 0, 0])
    lse, before = torch.zeros(3, 4, device="cuda"), c.weights.clone()
    out = ops.paged_attn(queries(c, 2), c.kv, c.table, c.lens, weights=c.weights, lse=lse)
    assert torch.all(out == 0) and torch.all(torch.isneginf(lse))
    assert torch.equal(c.weights.nan_to_num(), before.nan_to_num())


def test_attention_follows_the_formula_for_infinities_and_nan():
    c = Cache(4, 1, 64, 16, 20, BF16, seed=8, lens=[300, 300, 300, 300])
    q = torch.ones(4, 1, 1, 64, dtype=BF16, device="cuda")
    def put(s, i, plane, value):
        c.kv[plane, int(c.table_h[s, i // 16]), 0, i % 16] = value
    put(0, 299, 0, float("-inf"))           # weight 0: as if the token were not there
    put(1, 5, 0, float("inf"))              # inf - inf
    put(2, 130, 1, float("inf"))            # a value is infinite
    put(3, 200, 0, float("nan"))
    out = ops.paged_attn(q, c.kv, c.table, c.lens).float()
    short = c.lens.clone()
    short[0] = 299
    assert torch.equal(out[0], ops.paged_attn(q, c.kv, c.table, short).float()[0]) or \
        torch.allclose(out[0], ops.paged_attn(q, c.kv, c.table, short).float()[0], rtol=2 ** -7, atol=2 ** -9)
    assert torch.all(torch.isnan(out[1]))
    assert torch.all(torch.isinf(out[2]))
    assert torch.all(torch.isnan(out[3]))


def test_attention_repeats_bit_for_bit_and_adds_weights_up():
    c = Cache(5, 4, 128, 64, 40, BF16, seed=9, lens=[2500, 1, 0, 777, 64])
    q = queries(c, 8)
    first = ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights)
    once = c.weights.clone()
    c.weights.copy_(torch.from_numpy(c.w64).float())
    again = ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights)
    assert torch.equal(first, again) and torch.equal(once.nan_to_num(), c.weights.nan_to_num())
    assert torch.equal(first, ops.paged_attn(q, c.kv, c.table, c.lens))


def test_sessions_may_share_pages_they_read():
    c = Cache(2, 2, 64, 16, 8, BF16, seed=10, lens=[128, 128])
    c.table[1] = c.table[0]
    c.table64 = c.table.cpu().numpy()
    q = queries(c, 2)
    before = c.w64.copy()
    out = ops.paged_attn(q, c.kv, c.table, c.lens, weights=c.weights)
    check_attention(c, q, out, None, before, c.weights)


def test_bad_pages_and_counts_are_reported():
    c = Cache(3, 2, 64, 16, 8, BF16, seed=11, lens=[100, 100, 100])
    q = queries(c, 1)
    good = ops.paged_attn(q, c.kv, c.table, c.lens)
    ops.check_status(torch.device("cuda"))
    for page in (-1, c.kv.shape[1], 2 ** 31 - 1):
        table = c.table.clone()
        table[1, 3] = page
        out = ops.paged_attn(q, c.kv, table, c.lens)
        with pytest.raises(RuntimeError, match="page"):
            ops.check_status(torch.device("cuda"))
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    for n in (-1, 129, 2 ** 31 - 1):
        lens = c.lens.clone()
        lens[1] = n
        out = ops.paged_attn(q, c.kv, c.table, lens)
        with pytest.raises(RuntimeError, match="page"):
            ops.check_status(torch.device("cuda"))
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("Dh,page,T,nhd", [(128, 16, 1, False), (64, 32, 7, True), (128, 64, 300, False), (64, 256, 65, False)])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("with_weights", [False, True])
def test_append(Dh, page, T, nhd, padded, with_weights):
    lens = [[0, 3], [15, 16], [40, 0]]
    c = Cache(3, 2, Dh, page, -(-(40 + 2 * T) // page), BF16, seed=T, lens=lens, nhd=nhd)
    n_new = torch.tensor([T, 0, max(0, T - 2)], dtype=torch.int32) if padded else None
    for step in range(2):
        (k, v, w), (k64, v64, w64) = c.new(T, seed=20 + step, with_weights=with_weights)
        ops.paged_append_(c.kv, c.table, c.lens, c.next_pos, k, v, None if n_new is None else n_new.cuda(), c.weights,
                          c.positions, w)
        paged_oracle.append(c.kv64, c.table64, c.lens64, c.next64, k64, v64, n_new, c.w64, c.pos64, w64)
    c.assert_same_state()


def test_append_without_weights_and_into_other_counts():
    c = Cache(2, 3, 64, 16, 4, F16, seed=3, lens=[5, 20])
    (k, v, _), (k64, v64, _) = c.new(9, seed=4)
    lens, next_pos = torch.empty_like(c.lens), torch.empty_like(c.next_pos)
    w, pos = c.weights.clone(), c.positions.clone()
    ops.paged_append_(c.kv, c.table, c.lens, c.next_pos, k, v, lens_out=lens, next_pos_out=next_pos)
    assert torch.equal(c.lens.cpu(), c.lens_h) and torch.equal(c.next_pos.cpu(), c.next_h)
    assert torch.equal(w.nan_to_num(), c.weights.nan_to_num()) and torch.equal(pos, c.positions)
    paged_oracle.append(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64.copy(), c.pos64.copy())
    assert np.array_equal(lens.cpu().numpy(), c.lens64) and np.array_equal(next_pos.cpu().numpy(), c.next64)
    assert np.array_equal(c.kv.double().cpu().numpy(), c.kv64, equal_nan=True)


def test_append_of_nothing_changes_nothing():
    c = Cache(2, 2, 64, 16, 4, F16, seed=3, lens=[5, 20])
    (k, v, _), _ = c.new(4, seed=4)
    ops.paged_append_(c.kv, c.table, c.lens, c.next_pos, k[:, :, :0], v[:, :, :0], weights=c.weights, positions=c.positions)
    ops.paged_append_(c.kv, c.table, c.lens, c.next_pos, k, v, torch.zeros(2, dtype=torch.int32, device="cuda"), c.weights,
                      c.positions)
    c.assert_same_state()


def test_append_drops_and_reports_what_has_no_room():
    c = Cache(2, 2, 64, 16, 2, F16, seed=3, lens=[30, 3])
    (k, v, _), (k64, v64, _) = c.new(5, seed=4)
    ops.paged_append_(c.kv, c.table, c.lens, c.next_pos, k, v, weights=c.weights, positions=c.positions)
    paged_oracle.append(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64)
    c.assert_same_state()
    with pytest.raises(RuntimeError, match="page"):
        ops.check_status(torch.device("cuda"))


# ------------------------------------------------------------------------------------------------ under a budget
@pytest.mark.parametrize("lens,T,keep,sink,recent", [
    ([50, 50], 1, 50, 4, 10),             # at the budget, one more
    ([50, 31], 16, 50, 0, 0),             # nothing shielded: new tokens without weight go first
    ([0, 3], 9, 50, 2, 8),                # below the budget: a plain append
    ([45, 49], 9, 50, 2, 8),              # reaches the budget within the call
    ([0, 10], 200, 50, 4, 20),            # a prompt longer than the budget
    ([90, 70], 3, 50, 1, 49),             # the budget was lowered; everything kept is shielded
    ([90, 50], 0, 50, 1, 9),              # ... with nothing new
    ([1, 0], 1, 1, 0, 1),                 # a budget of one
    ([1, 1], 5, 1, 0, 0)])
@pytest.mark.parametrize("Dh,page", [(64, 16), (128, 32)])
@pytest.mark.parametrize("with_weights", [False, True])
def test_append_under_a_budget(lens, T, keep, sink, recent, Dh, page, with_weights):
    c = Cache(2, 3, Dh, page, -(-(max(lens + [keep])) // page) + 1, BF16, seed=sum(lens) + T, lens=lens)
    for step in range(3):
        (k, v, w), (k64, v64, w64) = c.new(T, seed=30 + step, with_weights=with_weights)
        ops.paged_append_evict_(c.kv, c.table, c.lens, c.next_pos, k, v, c.weights, c.positions, keep, sink, recent, w_new=w)
        paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, keep, sink, recent, w64)
        c.assert_same_state()


@pytest.mark.parametrize("S,H,lens,T,keep,sink,recent", [
    (1, 2, [4096], 1, 4096, 4, 64), (2, 1, [5000, 4999], 300, 5000, 16, 1000), (1, 1, [20000], 1000, 20000, 0, 0),
    (1, 1, [100], 9000, 777, 10, 100), (1, 2, [40000], 17, 33333, 4, 16),
    (1, 2, [40000], 3, 9000, 4, 16), (1, 1, [20000], 3, 40, 2, 8)])       # budgets lowered by much
def test_long_budgets(S, H, lens, T, keep, sink, recent):
    c = Cache(S, H, 64, 64, -(-max(lens + [keep]) // 64), F16, seed=T, lens=lens)
    for step in range(2):
        (k, v, w), (k64, v64, w64) = c.new(T, seed=40 + step, with_weights=True)
        ops.paged_append_evict_(c.kv, c.table, c.lens, c.next_pos, k, v, c.weights, c.positions, keep, sink, recent, w_new=w)
        paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, keep, sink, recent, w64)
        c.assert_same_state()


@pytest.mark.parametrize("S,H,keep,T", [(100, 3, 5300, 9), (40, 2, 11000, 50), (3, 1, 70001, 3)])
def test_a_session_does_not_depend_on_its_batch(S, H, keep, T):
    # many heads: small CTAs that go through their candidates in rounds; one session alone: larger ones, or a cluster
    page, Dh = 64, 64
    M = -(-keep // page)
    g = torch.Generator(device="cuda").manual_seed(S)
    table = torch.randperm(S * M, generator=g, device="cuda").view(S, M).int()
    kv = torch.randn(2, S * M, H, page, Dh, generator=g, device="cuda", dtype=BF16)
    weights = torch.rand(S * M, H, page, generator=g, device="cuda").mul_(64).floor_()           # a few values: many ties
    positions = torch.randint(0, 2 * keep, (S * M, H, page), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.full((S, H), keep, dtype=torch.int32, device="cuda")
    next_pos = torch.full((S, H), 2 * keep, dtype=torch.int32, device="cuda")
    new = torch.randn(2, S, H, T, Dh, generator=g, device="cuda", dtype=BF16)
    w_new = torch.rand(S, H, T, generator=g, device="cuda") * 64
    both = [[x.clone() for x in (kv, lens, next_pos, weights, positions)] for _ in range(2)]
    a, b = both
    ops.paged_append_evict_(a[0], table, a[1], a[2], new[0], new[1], a[3], a[4], keep, 5, keep // 50, w_new=w_new)
    for s in range(S):
        ops.paged_append_evict_(b[0], table[s:s + 1], b[1][s:s + 1], b[2][s:s + 1], new[0, s:s + 1], new[1, s:s + 1], b[3], b[4],
                                keep, 5, keep // 50, w_new=w_new[s:s + 1])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.all(a[1] == keep) and torch.all(a[2] == 2 * keep + T) and not torch.equal(a[4], positions)


@pytest.mark.parametrize("padded", [[3, 0, 7], [0, 0, 0], [7, 7, 1]])
def test_padded_batch_under_a_budget(padded):
    c = Cache(3, 2, 64, 16, 5, BF16, seed=9, lens=[[60, 64], [64, 64], [10, 61]], nhd=True)
    n_new = torch.tensor(padded, dtype=torch.int32)
    (k, v, w), (k64, v64, w64) = c.new(7, seed=1, with_weights=True)
    ops.paged_append_evict_(c.kv, c.table, c.lens, c.next_pos, k, v, c.weights, c.positions, 64, 3, 8, n_new.cuda(), w)
    paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, n_new, c.w64, c.pos64, 64, 3, 8, w64)
    c.assert_same_state()


@pytest.mark.parametrize("value", [0.0, -0.0, 1.0, float("inf"), float("-inf"), float("nan"), 1e-45])
def test_eviction_among_equal_and_odd_weights(value):
    # every weight the same: the lowest indexes are kept; then a few others among them
    for others in ([], [0.0, -1.0, 2.0, float("inf"), float("nan"), float("-inf"), -0.0, 1e-40]):
        c = Cache(1, 1, 64, 16, 10, BF16, seed=12, lens=[150])
        pg = torch.from_numpy(c.table64[0].copy()).long()
        w = torch.full((160,), value)
        for j, x in enumerate(others):
            w[7 + 11 * j] = x
        w[150:] = float("nan")
        c.weights[pg.cuda(), 0] = w.view(10, 16).cuda()
        c.w64[pg.numpy(), 0] = w.double().view(10, 16).numpy()
        (k, v, w_new), (k64, v64, w64) = c.new(4, seed=2, with_weights=True)
        ops.paged_append_evict_(c.kv, c.table, c.lens, c.next_pos, k, v, c.weights, c.positions, 140, 3, 5, w_new=w_new)
        paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, 140, 3, 5, w64)
        c.assert_same_state()


# ------------------------------------------------------------------------------------------------ together
def test_sessions_under_a_budget_decode_step_by_step():
    """Prompt, then steps of append, attention with weights, eviction; attention against 64 bits at every step, and the
    state moved by the host's rules from the device's own weights."""
    S, H, G, Dh, page, keep = 3, 2, 2, 64, 16, 48
    c = Cache(S, H, Dh, page, 4, BF16, seed=1, lens=[0, 0, 0])
    slab = PagedSlab(S, H, Dh, BF16, page, 40, 64, keep=keep, sink=2, recent=8)
    for s in range(S):
        slab.reserve(s, keep)
    c.kv, c.weights, c.positions = slab.kv, slab.weights, slab.positions
    c.table, c.lens, c.next_pos = slab.table, slab.lens, slab.next_pos
    c.kv64, c.w64, c.pos64 = slab.kv.double().cpu().numpy(), slab.weights.double().cpu().numpy(), slab.positions.cpu().numpy()
    c.table64, c.lens64, c.next64 = slab.table.cpu().numpy(), slab.lens.cpu().numpy(), slab.next_pos.cpu().numpy()
    (k, v, _), (k64, v64, _) = c.new(40, seed=70)
    n_new = torch.tensor([40, 17, 0], dtype=torch.int32)
    slab.append(k, v, n_new.cuda())
    paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, n_new, c.w64, c.pos64, keep, 2, 8)
    c.assert_same_state()
    for step in range(30):
        (k, v, _), (k64, v64, _) = c.new(1, seed=80 + step)
        q = queries(c, G, seed=step)
        out = slab.append_and_attend(q, k, v)
        paged_oracle.append_evict(c.kv64, c.table64, c.lens64, c.next64, k64, v64, None, c.w64, c.pos64, keep, 2, 8)
        before = c.w64.copy()
        c.assert_same_state(weights_exact=False)
        check_attention(c, q, out, None, before, slab.weights)
        c.w64 = slab.weights.double().cpu().numpy()          # the next eviction goes by the device's own sums


def test_a_captured_step_replays_across_the_budget():
    S, H, Dh, page, keep = 2, 2, 128, 16, 20
    def slab():
        x = PagedSlab(S, H, Dh, BF16, page, 8, 32, keep=keep, sink=1, recent=4)
        for s in range(S):
            x.reserve(s, keep)
        return x
    eager, graphed = slab(), slab()
    g = torch.Generator().manual_seed(5)
    steps = [[torch.randn(S, n, 1, Dh, generator=g).to(BF16).cuda() for n in (4 * H, H, H)] for _ in range(30)]
    held = [torch.empty_like(t) for t in steps[0]]
    warm = slab()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.append_and_attend(*held)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                       # two graphs of the same step, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = graphed.append_and_attend(*held)
        graphs.append((graph, y))
    for i, step in enumerate(steps):
        want = eager.append_and_attend(*step)
        for a, b in zip(held, step):
            a.copy_(b)
        graph, y = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
    for name in ("kv", "weights", "positions", "lens", "next_pos"):
        assert torch.equal(getattr(eager, name), getattr(graphed, name)), name


def test_a_step_of_everything_on_two_streams():
    """Two slabs of their own, a step of each on a stream of its own, over and over: as one after the other."""
    def slab():
        x = PagedSlab(6, 4, 128, BF16, 32, 6 * 20, 640, keep=600, sink=4, recent=50)
        for s in range(6):
            x.reserve(s, 600)
        return x
    g = torch.Generator().manual_seed(3)
    prompt = torch.randn(2, 6, 4, 590, 128, generator=g).to(BF16).cuda()
    steps = [[torch.randn(6, n, 1, 128, generator=g).to(BF16).cuda() for n in (8, 4, 4)] for _ in range(25)]
    alone = slab()
    alone.append(prompt[0], prompt[1])
    want = [alone.append_and_attend(*x) for x in steps]
    torch.cuda.synchronize()
    pair, got = [slab(), slab()], [[], []]
    streams = [torch.cuda.Stream() for _ in pair]
    torch.cuda.synchronize()
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            pair[i].append(prompt[0], prompt[1])
    for x in steps:
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(pair[i].append_and_attend(*x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want))
        for name in ("kv", "weights", "positions", "lens", "next_pos"):
            assert torch.equal(getattr(pair[i], name), getattr(alone, name)), name


def test_calls_on_two_streams_do_not_disturb_each_other():
    caches = [Cache(4, 4, 128, 32, 40, BF16, seed=50 + i, lens=[1200, 5, 300, 1280]) for i in range(2)]
    qs = [queries(c, 4, seed=i) for i, c in enumerate(caches)]
    want = [ops.paged_attn(q, c.kv, c.table, c.lens) for c, q in zip(caches, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.paged_attn(qs[i], caches[i].kv, caches[i].table, caches[i].lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("budget", [dict(), dict(keep=20, sink=1, recent=4)])
def test_traces_as_one_graph(budget):
    slab = PagedSlab(2, 2, 64, BF16, 16, 8, 32, **budget)
    ref = PagedSlab(2, 2, 64, BF16, 16, 8, 32, **budget)
    for s in range(2):
        slab.reserve(s, 30)
        ref.reserve(s, 30)
    step = torch.compile(lambda q, k, v: slab.append_and_attend(q * 2, k, v) + 1, fullgraph=True, backend="aot_eager")
    g = torch.Generator().manual_seed(6)
    for _ in range(25):
        q, k, v = (torch.randn(2, n, 1, 64, generator=g).to(BF16).cuda() for n in (4, 2, 2))
        with torch.no_grad():
            assert torch.equal(step(q, k, v), ref.append_and_attend(q * 2, k, v) + 1)
    assert torch.equal(slab.weights, ref.weights) and torch.equal(slab.kv, ref.kv)


def test_sessions_take_and_give_back_pages():
    slab = PagedSlab(2, 1, 64, BF16, 16, 3, 48)
    slab.reserve(0, 33)
    assert slab.free_pages == 0 and slab.room(0) == 48
    with pytest.raises(RuntimeError, match="free pages"):
        slab.reserve(1, 1)
    k = torch.randn(2, 1, 33, 64, device="cuda").to(BF16)
    slab.append(k, k, torch.tensor([33, 0], dtype=torch.int32, device="cuda"))
    q = torch.randn(2, 1, 1, 64, device="cuda").to(BF16)
    assert torch.all(slab.attend(q)[1] == 0)
    slab.release(0)
    slab.reserve(1, 16)
    slab.append(k[:, :, :16], k[:, :, :16], torch.tensor([0, 16], dtype=torch.int32, device="cuda"))
    y = slab.attend(q)
    assert torch.all(y[0] == 0) and not torch.any(torch.isnan(y)) and torch.any(y[1] != 0)
    slab.append(k[:, :, :1], k[:, :, :1], torch.tensor([1, 0], dtype=torch.int32, device="cuda"))      # has no page
    with pytest.raises(RuntimeError, match="page"):
        ops.check_status(torch.device("cuda"))
