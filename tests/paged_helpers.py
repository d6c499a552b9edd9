"""Caches and tolerances of the paged cache tests."""
import numpy as np
import torch

from oracle import paged_oracle


class Cache:
    """A paged cache on the device with its 64-bit twin on the host; every slot no session holds is NaN."""

    def __init__(self, S, H, Dh, page, M, dtype, seed=0, lens=None, nhd=False, spare=3, k_gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.S, self.H, self.Dh, self.page, self.M = S, H, Dh, page, M
        P = S * M + spare
        self.table_h = torch.randperm(P, generator=g)[:S * M].view(S, M).int()
        lens = torch.zeros(S, H, dtype=torch.int32) if lens is None else torch.as_tensor(lens, dtype=torch.int32)
        self.lens_h = lens.expand(S, H) if lens.dim() == 2 else lens[:, None].expand(S, H)
        self.lens_h = self.lens_h.contiguous().clone()
        kv = torch.randn(2, P, H, page, Dh, generator=g).to(dtype).float()
        kv[0] *= k_gain
        kv = kv.to(dtype).float()
        weights = torch.rand(P, H, page, generator=g) ** 4
        weights[torch.rand(P, H, page, generator=g) < 0.1] = 0.0            # ties
        held = torch.zeros(P, H, page, dtype=torch.bool)
        positions = torch.full((P, H, page), -5, dtype=torch.int32)
        self.next_h = torch.zeros(S, H, dtype=torch.int32)
        for s in range(S):
            for h in range(H):
                n = int(self.lens_h[s, h])
                i = torch.arange(n)
                pg, row = self.table_h[s, i // page].long(), i % page
                held[pg, h, row] = True
                pos = torch.randperm(2 * n + 1, generator=g)[:n].int()      # any distinct positions, any order
                positions[pg, h, row] = pos
                self.next_h[s, h] = 2 * n + 1
        kv[:, ~held] = float("nan")
        weights[~held] = float("nan")
        # device
        if nhd:      # pages as [page, H, Dh]
            self.kv = torch.empty(2, P, page, H, Dh, dtype=dtype, device="cuda").transpose(2, 3)
            self.kv.copy_(kv)
        else:
            self.kv = kv.to(dtype).cuda()
        self.weights, self.positions = weights.cuda(), positions.cuda()
        self.table, self.lens, self.next_pos = self.table_h.cuda(), self.lens_h.cuda(), self.next_h.cuda()
        # host
        self.kv64, self.w64, self.pos64 = kv.double().numpy(), weights.double().numpy(), positions.numpy().copy()
        self.table64, self.lens64, self.next64 = self.table_h.numpy(), self.lens_h.numpy().copy(), self.next_h.numpy().copy()
        self.dtype = dtype

    def new(self, T, seed, with_weights=False):
        g = torch.Generator().manual_seed(seed)
        new = torch.randn(self.S, T, 2, self.H, self.Dh, generator=g).to(self.dtype)
        k, v = new[:, :, 0].transpose(1, 2), new[:, :, 1].transpose(1, 2)
        w = torch.rand(self.S, self.H, T, generator=g) ** 4 if with_weights else None
        dev = new.cuda()
        return ((dev[:, :, 0].transpose(1, 2), dev[:, :, 1].transpose(1, 2), None if w is None else w.cuda()),
                (k.double().numpy(), v.double().numpy(), None if w is None else w.double().numpy()))

    def assert_same_state(self, weights_exact=True):
        """Everything is moved, nothing computed: the device state must be the host's, bit for bit."""
        torch.cuda.synchronize()
        assert np.array_equal(self.lens.cpu().numpy(), self.lens64)
        assert np.array_equal(self.next_pos.cpu().numpy(), self.next64)
        assert np.array_equal(self.positions.cpu().numpy(), self.pos64)
        assert np.array_equal(self.kv.double().cpu().numpy(), self.kv64, equal_nan=True)
        if weights_exact:
            assert np.array_equal(self.weights.double().cpu().numpy(), self.w64, equal_nan=True)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_attention(c, q, out, lse=None, weights_before=None, weights_after=None, scale=None):
    """The kernel against softmax attention in 64 bits.

    A logit is a sum of Dh products held in fp32: its error is at most Dh * 2^-23 of sum |q||k| (truncating adds count
    a whole step each), times the scale; e^x turns it into a relative error of the same size, and normalising doubles it.
    Scaling and 2^x add a few fp32 steps of the exponent's argument (|x| log2 e <= 2^8 here) and 2^-21 of the result: far
    below.  The weight of a token is rounded to 16 bits once for the product with v (half a step of each p |v|; values
    below the normal range of fp16 by at most 2^-25 of the largest weight, which is at least 2^-8 of the sum's scale),
    the result once more.  Partial results are held and joined in fp32."""
    q64 = q[:, :, 0].double().cpu().numpy()
    want, want_lse, given, spread = paged_oracle.attend(q64, c.kv64, c.table64, c.lens64, scale)
    G = q64.shape[1] // c.H
    u = half_step(c.dtype)
    sc = c.Dh ** -0.5 if scale is None else scale
    dx = np.zeros(want_lse.shape)
    vmax = np.zeros(want_lse.shape)
    for s in range(c.S):
        for h in range(c.H):
            n = int(c.lens64[s, h])
            if n:
                i = np.arange(n)
                pg, row = c.table64[s, i // c.page], i % c.page
                qk = np.abs(q64[s, h * G:(h + 1) * G]) @ np.abs(c.kv64[0, pg, h, row]).T
                dx[s, h * G:(h + 1) * G] = (c.Dh * 2.0 ** -23 * sc * qk).max(axis=1)
                vmax[s, h * G:(h + 1) * G] = n * np.abs(c.kv64[1, pg, h, row]).max()
    tol = (u + 2 * dx[..., None] + 2.0 ** -18) * spread + u * np.abs(want)
    if c.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * vmax[..., None] + 2.0 ** -25
    got = out[:, :, 0].double().cpu().numpy()
    assert np.all(np.isfinite(got))
    worst = np.max(np.abs(got - want) / np.maximum(tol, 1e-300))
    assert worst <= 1.0, f"output off by {worst} of the tolerance"
    if lse is not None:
        d = np.abs(np.nan_to_num(lse.double().cpu().numpy(), neginf=-1e30) - np.nan_to_num(want_lse, neginf=-1e30))
        bound = dx + 2.0 ** -18 + 2.0 ** -22 * np.abs(np.nan_to_num(want_lse, neginf=-1e38))
        assert np.all(d <= bound), f"lse off by {np.max(d / bound)} of the tolerance"
    if weights_after is not None:
        # dx above is the largest of a head; a token's weight adds G terms and one fp32 sum
        w = weights_before.copy()
        paged_oracle.add_given(w, c.table64, given, c.page)
        got = weights_after.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(w))
        rel = 2 * dx.max() + (G + 4) * 2.0 ** -23 + 2.0 ** -18
        added = np.where(np.isnan(w), 0.0, w - weights_before)
        bound = rel * added + 2.0 ** -23 * np.abs(np.nan_to_num(w)) + 1e-30
        d = np.abs(np.nan_to_num(got) - np.nan_to_num(w))
        assert np.all(d <= bound), f"weights off by {np.max(d / bound)} of the tolerance"
