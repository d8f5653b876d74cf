"""Buckets of relative positions, on the host, against their definition in whole numbers."""
from fractions import Fraction

import pytest
import torch


@pytest.mark.parametrize("buckets,far", [(32, 128), (4, 2), (4, 64), (8, 3), (20, 160), (40, 320), (60, 480), (108, 64), (120, 960), (16, 1000), (32, 9)])
def test_buckets_by_distance(buckets, far):
    from savit_amd import ops

    N = far + 5
    index, n = ops.relpos_index_1d(N, buckets, far, device="cpu")
    assert n == buckets and index.dtype == torch.int32 and index.shape == (N, N)
    half, near = buckets // 2, buckets // 4
    want = []
    for a in range(N):
        if a < near:
            want.append(a)
            continue
        k = 0  # the k-th logarithmic bucket begins at near (far / near)^(k / (half - near))
        while k + 1 < half - near and Fraction(a, near) ** (half - near) >= Fraction(far, near) ** (k + 1):
            k += 1
        want.append(near + k)
    assert index[0, 1:].tolist() == [half + w for w in want[1:]] and index[:, 0].tolist() == want
    d = torch.arange(N)[None, :] - torch.arange(N)[:, None]
    assert torch.equal(index.long(), torch.tensor(want)[d.abs()] + half * (d > 0).long())
