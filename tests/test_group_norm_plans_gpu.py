"""Group norm where its sums are longest: 32 pieces per thread in one pass, hundreds of chunks, groups of hundreds and thousands of
channels.  Values and bounds are those of test_group_norm_gpu.reference; what a sum of 32-bit terms loses, E x 2^-24 of the
magnitudes it adds, is counted here from the plan that the call takes (`sums`), not taken as a constant."""
import math

import pytest
import torch

import test_group_norm_gpu as base

pytestmark = pytest.mark.gpu


def log2(n):
    return math.ceil(math.log2(max(n, 1)))


def sums(shape, G, elem, backward):
    """roundings along the longest way of a term into a group's or a channel's sum (csrc/norm_ops.hip, gn_plan and its kernels)"""
    N, C = shape[0], shape[-1]
    P = math.prod(shape[1:-1])
    Cg, V = C // G, 16 // elem
    while C % V:
        V //= 2
    for k in range(1, G + 1):
        sc = k * Cg
        if G % k or sc % V or (sc * elem < 64 and k < G):
            continue
        if sc // V > 512:
            break
        pieces = math.ceil(P / (512 // (sc // V)))
        if pieces > (16 if backward else 32):
            break
        # pieces in a row, the V elements of an access, lanes and waves or trees over rows and channels, samples in a row
        return "slab", pieces + V + 9 + 8 + log2(Cg) + N
    cv = C // V
    RP = 256 // cv if cv < 256 else 1
    unit = 8 * RP
    rows = math.ceil(math.ceil(P / unit) / math.ceil(2048 / N)) * unit
    chunks = math.ceil(P / rows)
    if not backward:
        # eight rows in a row, then merges of (count, mean, deviations) at four roundings each: a thread's groups of eight, rows side
        # by side, channels of the group, a thread's list of chunks, lanes and waves
        return "two passes", 8 + 4 * (rows // unit + log2(RP) + log2(Cg) + math.ceil(chunks / 256) + 6 + 3)
    J = 1 if Cg >= 256 else 256 // Cg
    last = max(math.ceil(Cg / (256 // J)) + 8, N)                          # the group's channels, or the samples
    if math.ceil(chunks / J) > 64:
        J, last = 32, max(math.ceil(Cg / 256) + 8, N)
    # a thread's rows, rows side by side, a list of chunks, the lists
    return "two passes", rows // RP + log2(RP) + math.ceil(chunks / J) + log2(J) + last


CASES = [((1, 2000, 256), 4, "slab", "two passes"), ((1, 6000, 2048), 1, "two passes", "two passes"), ((1, 6000, 2048), 8, "two passes", "two passes"),
         ((1, 25088, 512), 1, "two passes", "two passes"), ((1, 700, 8192), 2, "two passes", "two passes"), ((3, 9000, 300), 1, "two passes", "two passes")]


@pytest.mark.parametrize("shape,G,fwd,bwd", CASES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_long_sums(shape, G, fwd, bwd, dt, monkeypatch):
    elem = torch.finfo(dt).bits // 8
    f, b = sums(shape, G, elem, False), sums(shape, G, elem, True)
    if dt == torch.bfloat16:
        assert (f[0], b[0]) == (fwd, bwd)
    monkeypatch.setattr(base, "E", max(f[1], b[1]) * base.F)
    base.run_case(shape, G, "relu" if G == 8 else None, dt, seed=5)
