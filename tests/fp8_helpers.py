"""Pools, batches and error bounds shared by the tests of the 8-bit paged cache."""

from __future__ import annotations

import numpy as np
import torch

from barellm_b200 import ops
from oracle import fp8_oracle as f8

STALE = 0x7F  # NaN code: a stale slot that reaches an output shows


class Pool:
    """An 8-bit pool on the host (oracle) and on the device, with shuffled blocks."""

    def __init__(self, device, layers, blocks, hkv, bs, d, fill=STALE, seed=0):
        shape = (layers, blocks, hkv, bs, d)
        self.codes = [np.full(shape, fill, dtype=np.uint8) for _ in range(2)]
        self.scales = [np.full(shape[:3], 1.0, dtype=np.float32) for _ in range(2)]
        self.dev = [torch.from_numpy(c.copy()).to(device).view(ops.FP8_DTYPE) for c in self.codes]
        self.dev_scales = [torch.from_numpy(s.copy()).to(device) for s in self.scales]
        self.free = np.random.RandomState(seed).permutation(blocks).tolist()
        self.bs, self.device = bs, device

    @property
    def args(self):
        return (*self.dev, *self.dev_scales)

    def table(self, n_tokens):
        """Block tables for rows that will hold ``n_tokens`` each, padded with -1."""
        nb = [-(-n // self.bs) for n in n_tokens]
        t = np.full((len(nb), max(1, max(nb))), -1, dtype=np.int32)
        for i, n in enumerate(nb):
            t[i, :n] = [self.free.pop() for _ in range(n)]
        return t

    def assert_equal(self):
        for c, s, dc, ds in zip(self.codes, self.scales, self.dev, self.dev_scales):
            np.testing.assert_array_equal(dc.view(torch.uint8).cpu().numpy(), c)
            np.testing.assert_array_equal(ds.cpu().numpy(), s)

    def download(self):
        """The device's pool as the oracle's."""
        self.codes = [c.view(torch.uint8).cpu().numpy() for c in self.dev]
        self.scales = [s.cpu().numpy() for s in self.dev_scales]


def i32(values, device):
    return torch.tensor(list(values), dtype=torch.int32, device=device)


def cache_values(rs, h, n, d, spread=0.5):
    """Token magnitudes and a few channels vary, as in a model's K and V."""
    return (rs.randn(h, n, d) * np.exp(spread * rs.randn(h, 1, d)) * np.exp(spread * rs.randn(h, n, 1))).astype(np.float32)


def filled(device, lens, hkv, bs, d, dtype, seed=0, layers=2, layer=1, spread=0.5):
    """A pool whose rows hold ``lens`` tokens (appended by the kernel), and their table."""
    rs = np.random.RandomState(seed)
    blocks = sum(-(-n // bs) for n in lens) + 5
    pool = Pool(device, layers, blocks, hkv, bs, d, seed=seed)
    table = pool.table(lens)
    bt = torch.from_numpy(table).to(device)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    if off[-1]:
        k = torch.from_numpy(cache_values(rs, hkv, int(off[-1]), d, spread)).to(dtype).to(device).unsqueeze(0)
        v = torch.from_numpy(cache_values(rs, hkv, int(off[-1]), d, spread)).to(dtype).to(device).unsqueeze(0)
        ops.paged_append_fp8(*pool.args, layer, bt, i32([0] * len(lens), device), k, v,
                             new_offsets=torch.from_numpy(off).to(device), max_new_tokens=max(lens))
    pool.download()
    return pool, table, bt


def attention_bound(out, spread, reach, flat, q, dtype, weight_eps, keys):
    """Largest error the kernels' arithmetic can leave in ``out`` [H, C, D].

    A score is an fp32 sum of D products: D + 8 roundings (products and sums, the
    scale factors, the exponent's argument) move it by at most (D + 8) 2^-24
    ``reach``.  q in fp16, its largest element in [1, 2), keeps an element below
    2^-14 to half a step of 2^-24 of that range: 2^-25 ``flat`` more (a 16-bit q's
    other elements are exact).  An exponential adds 2^-21.  A relative error e
    of every weight moves out by at most 2 e spread (numerator and
    denominator).  ``weight_eps``: half a step of the type that holds P (0 where
    it stays fp32), in the numerator only.  The P V sum and the joins are fp32:
    (keys + 64) 2^-24 spread.  Last, half a step of the output and two of the
    fp32 division's."""
    d = q.shape[-1]
    delta = (reach * (d + 8) * 2.0 ** -24 + flat * 2.0 ** -25)[..., None] + 2.0 ** -21
    err = spread * (weight_eps + 2 * np.expm1(2 * delta) + (keys + 64) * 2.0 ** -24)
    half = torch.finfo(dtype).eps / 2
    return err + half * (np.abs(out) + err) + 2.0 ** -22 * np.abs(out) + float(torch.finfo(dtype).tiny)


def assert_within(got, want, bound):
    """Every value within its bound; NaN exactly where the definition has NaN (an infinite q)."""
    bad = np.where(np.isnan(want), ~np.isnan(got), ~(np.abs(got - want) <= bound))
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(got - want) / bound)), np.argwhere(bad)[:4].tolist())
