"""Packed batches: ragged sequences laid end to end, the form the GatedDeltaNet kernels take through cu_seqlens,
for the rotary positions (``ops.qk_rope_fwd``) and the attention core (``ops.attn_packed_fwd``).

``PackedPlan`` holds one batch's geometry on the device: each token's position in its sequence and the 128-token
block tables the attention kernels walk (r97b_packed_blocks)."""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import R97bError, R97bPacked, lib


class PackedPlan:
    """The geometry of a ragged batch: cu_seqlens (host ints, from 0; empty sequences allowed) on `device`. Keep it as
    long as calls that take it may run; it holds nothing of the tensors."""

    def __init__(self, cu_seqlens, device):
        cu64 = np.asarray(cu_seqlens, dtype=np.int64).reshape(-1)
        if len(cu64) < 1 or cu64[0] != 0 or (np.diff(cu64) < 0).any() or cu64[-1] > 0x7FFFFF00:
            raise R97bError("bad cu_seqlens")
        self.cu = np.ascontiguousarray(cu64, dtype=np.int32)
        self.lens = np.diff(self.cu)
        self.n_seq, self.T = len(self.cu) - 1, int(self.cu[-1])
        self.max_len = int(self.lens.max()) if self.n_seq else 0
        n = int(lib().r97b_packed_blocks(self.cu.ctypes.data, self.n_seq, None, None))
        if n < 0:
            raise R97bError("bad cu_seqlens")
        # one buffer, one copy: the two block tables, then the positions
        host = np.empty(8 * n + self.T, dtype=np.int32)
        lib().r97b_packed_blocks(self.cu.ctypes.data, self.n_seq, host[:4 * n].ctypes.data, host[4 * n:8 * n].ctypes.data)
        host[8 * n:] = np.arange(self.T, dtype=np.int32) - np.repeat(self.cu[:-1], self.lens)
        self.n_blocks = n
        self.buf = torch.from_numpy(host).to(device)
        self.device = self.buf.device
        self.pos = self.buf[8 * n:]
        base = self.buf.data_ptr()
        self._k_host = host[4 * n:8 * n].copy()
        self.desc = R97bPacked(self.n_seq, n, self.T, base, base + 16 * n, self._k_host.ctypes.data)
        self.ref = ctypes.byref(self.desc)
