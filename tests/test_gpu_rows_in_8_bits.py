"""Codes of rows in 8 bits are those of their definition, to the bit: code = e4m3(y / scale), the quotient a rounded one of 32 bits, a value half way between two codes to
the even one; scale = max(max |y| / 448, 2^-126) is the rounded product with the rounded 1 / 448."""

import pytest
import torch

from distdl_amd import nn

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def defined(y):
    """On the CPU, whose 32-bit division is rounded once."""
    y = y.detach().cpu().float()
    scale = (y.abs().amax(-1, keepdim=True) * torch.tensor(1 / 448)).clamp(min=2.0 ** -126)
    return (y / scale).clamp(-448, 448).to(torch.float8_e4m3fn), scale[..., 0]


def same(codes, scales, y):
    want, want_scales = defined(y)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))


def borders(tops, cols):
    """Rows of the largest elements ``tops``; the others next to, or at, what lies half way between two codes."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    half_way = (codes[1:] + codes[:-1]) / 2
    g = torch.Generator().manual_seed(cols)
    rows = []
    for top in tops:
        top = torch.tensor(top, dtype=torch.float32)
        scale = (top * torch.tensor(1 / 448)).clamp(min=2.0 ** -126)
        row = half_way[torch.randint(0, len(half_way), (cols,), generator=g)] * scale
        for _ in range(2):
            way = torch.randint(-1, 2, (cols,), generator=g)
            row = torch.where(way == 0, row, torch.nextafter(row, torch.where(way < 0, torch.tensor(0.0), torch.tensor(float("inf")))))
        row = row.clamp(max=top) * torch.where(torch.rand(cols, generator=g) < 0.5, -1.0, 1.0)
        row[cols // 3], row[cols // 2] = -0.0, top
        rows.append(row)
    return torch.stack(rows).cuda()


@pytest.mark.parametrize("cols", [5, 8, 100, 512, 1000, 1030, 2501, 4096, 8190, 16384])
def test_values_next_to_a_border(cols):
    g = torch.Generator().manual_seed(1)
    tops = (448 * torch.exp2(torch.randint(-20, 20, (30,), generator=g)) * (1 + torch.rand(30, generator=g))).tolist()
    y = borders(tops + [448.0, 1.0, 3.0e38, 2.0 ** -117, 6.1e-36, 5.3e-36, 5.27e-36, 1e-38, 1e-42, 2.0 ** -100, 7e-30], cols)
    same(*nn.quantize_rows(y), y)


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("rows,cols", [(3000, 512), (700, 2048), (2500, 3333), (600, 8192)])
def test_rows_as_they_come(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, cols, generator=g).to(dtype).cuda()
    same(*nn.quantize_rows(x), x)


@pytest.mark.parametrize("cols", [7, 512, 1000, 2048, 4097, 8192, 12345])
@pytest.mark.parametrize("residual", [False, True], ids=["alone", "residual"])
def test_codes_of_normalised_rows_are_those_of_the_rows(cols, residual):
    """float32: the rows that the norm returns are what its 8-bit form stands for, before any rounding."""
    g = torch.Generator().manual_seed(cols)
    x, r, w = (torch.randn(*s, generator=g).cuda() for s in ((2100, cols), (2100, cols), (cols,)))
    y = nn.rms_norm_shard(x, w, r)[0] if residual else nn.rms_norm_shard(x, w)
    codes, scales = nn.rms_norm_shard(x, w, r if residual else None, eight_bit=True)[:2]
    same(codes, scales, y)
