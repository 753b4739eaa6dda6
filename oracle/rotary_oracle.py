"""Norm and rotary positions in 64 bits, from the definition (test
infrastructure; no reference counterpart).  Rows are [..., H, D] with one
position per [...]."""
import torch


def pair_columns(rot, start, interleaved):
    i = torch.arange(rot // 2)
    a = start + (2 * i if interleaved else i)
    return a, a + (1 if interleaved else rot // 2)


def _turn(y, positions, frequencies, start, interleaved, amplitude, sign):
    if frequencies is None:
        return y.clone()
    a, b = pair_columns(2 * frequencies.numel(), start, interleaved)
    angle = (positions.double()[..., None] * frequencies.double())[..., None, :]
    c, s = amplitude * torch.cos(angle), sign * amplitude * torch.sin(angle)
    out = y.clone()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def forward(x, weight, positions, frequencies, eps=1e-6, start=0, interleaved=False, amplitude=1.0):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    return _turn(x, positions, frequencies, start, interleaved, amplitude, 1.0)


def backward(x, weight, dy, positions, frequencies, eps=1e-6, start=0, interleaved=False, amplitude=1.0):
    """(dx, dweight, size of dx's terms per row, size of dweight's terms): the sizes bound the
    rounding of a computation in fewer bits."""
    x, d = x.double(), _turn(dy.double(), positions, frequencies, start, interleaved, amplitude, -1.0)
    if weight is None:
        return d, None, d.abs().amax(-1, keepdim=True), None
    w = weight.double()
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    n = x * r
    dw = (d * n).flatten(0, -2)
    t = d * w * n
    dx = r * (d * w - n * t.mean(-1, keepdim=True))
    size = r * ((d * w).abs().amax(-1, keepdim=True) + n.abs().amax(-1, keepdim=True) * t.abs().mean(-1, keepdim=True))
    return dx, dw.sum(0), size, dw.abs().sum(0)
