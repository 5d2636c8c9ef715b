"""The arithmetic behind token_probs on the GPU: a weight far below the largest and the sum over a whole vocabulary keep the
bits of a single float32 operation."""
from __future__ import annotations

import pytest
import torch

import ytensor_amd as yt

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check(p, x, temperature):
    """Logits are multiples of 1/4, so that their differences are exact, and every eight neighbours hold the row's largest,
    so that no part of a sum is scaled when it is joined to another. What is left, with steps of 2^-23:
      a weight   the exponential one step, its correction's product half a step
      the sum    a weight's error at most, and three additions in 32 bits (the others are in 64), half a step each
      the rest   the quotient and the product, half a step each
    5.5 steps. (A weight without its correction is off by 11 steps at 30 below the largest; a sum in 32 bits by half a step
    for each of the 150 numbers that a thread adds.)"""
    temperature = torch.tensor(temperature, dtype=torch.float32).double()  # as the call takes it
    want = torch.softmax(x.double().cpu() / temperature, -1)
    there = want > 2.0 ** -120
    off = ((p.double().cpu() - want).abs()[there] / want[there]).max().item()
    print(f"off by {off * 2 ** 23:.2f} steps", flush=True)
    assert off <= 5.5 * 2.0 ** -23
    assert (p.cpu()[~there] <= 2.0 ** -119).all()


def with_tops(x, top):
    n = x.shape[-1]
    x[..., torch.arange(n // 8) * 8 + torch.arange(n // 8) % 8] = top
    return x


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,n", [(1, 151936), (1, 1 << 21), (192, 151936), (193, 160008), (192, 9000), (3, 5000)])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_weights_and_their_sum(dtype, rows, n, temperature):
    """Few rows (in parts) and many (a workgroup each, held in registers or read twice), down to 45 below the largest."""
    x = 7.0 * torch.randn(rows, n, generator=torch.Generator().manual_seed(n))
    x = with_tops((4 * x).round().clamp(-128, 52) / 4, 13.0).to(DT[dtype])
    check(yt.token_probs(x.cuda(), temperature), x, temperature)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 16, 192])
@pytest.mark.parametrize("low", [-0.25, -0.5, -1.5, -3.75, -6.25, -10.25])
def test_rows_of_two_values(dtype, rows, low):
    """The same rounding at every addition does not add up."""
    x = with_tops(torch.full((rows, 151936), low), 0.0).to(DT[dtype])
    check(yt.token_probs(x.cuda(), 1.0), x, 1.0)
