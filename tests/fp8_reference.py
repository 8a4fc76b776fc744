"""Plain statements of the E4M3 block-scaled operators for the tests: quantisation by its f32 formula, everything
after it in 64 bits."""
import math

import torch

BLOCK = 128


def up(n, m):
    return (n + m - 1) // m * m


def padded(x, rows, columns):
    out = torch.zeros(up(x.shape[0], rows), up(x.shape[1], columns), dtype=torch.float32)
    out[:x.shape[0], :x.shape[1]] = x.float()
    return out


def quantize(x, rows_of):
    """x [rows, columns] on the CPU -> codes (float8_e4m3fn) and scales of blocks of rows_of x 128."""
    full = padded(x, rows_of, BLOCK)
    tiles = full.view(full.shape[0] // rows_of, rows_of, full.shape[1] // BLOCK, BLOCK)
    largest = tiles.abs().amax((1, 3))
    scales = torch.maximum(largest / torch.tensor(448.0), torch.tensor(2.0 ** -126))
    scales = torch.where(torch.isfinite(largest), scales, torch.tensor(math.nan))
    codes = (tiles / scales[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.reshape(full.shape)[:x.shape[0], :x.shape[1]], scales


def values(codes, scales, rows_of):
    """What codes stand for, in 64 bits."""
    full = scales.double().repeat_interleave(rows_of, 0).repeat_interleave(BLOCK, 1)
    return codes.double() * full[:codes.shape[0], :codes.shape[1]]


def activation(gate, up_, kind, beta=4.0, linear_beta=25.0):
    sig = 1 / (1 + torch.exp(-gate))
    if kind == "swiglu":
        return gate * sig * up_
    return beta * torch.tanh(gate / beta) * sig * linear_beta * torch.tanh(up_ / linear_beta)


def experts(x, ids, weights, tables, kind):
    """tables: (codes, scales) of w1, w3, w2, each per expert on the CPU."""
    xv = values(*quantize(x, 1), 1)
    out = torch.zeros(xv.shape, dtype=torch.float64)
    for e in range(tables[0][0].shape[0]):
        token, rank = (ids == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        w1, w3, w2 = (values(c[e], s[e], BLOCK) for c, s in tables)
        act = activation(xv[token] @ w1.t(), xv[token] @ w3.t(), kind)
        down = values(*quantize(act.float(), 1), 1) @ w2.t()
        out.index_add_(0, token, down * weights[token, rank].double().unsqueeze(1))
    return out
