"""Shared by the tests of the operators on rows of float32 / float16 / bfloat16 matrices: matrices with padded rows, and error bounds from the number formats."""
import torch

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U32 = 2.0 ** -24      # half a step of float32, relative

def half_step(dtype): return torch.finfo(dtype).eps / 2

def matrix(g, rows, cols, dtype, pad=0, scale=1.0, first=0, device="cuda"):
    """[rows, cols] view with `pad` elements between rows and `first` elements in front of the first one; the space around it holds 77"""
    base = torch.full((rows * (cols + pad) + first,), 77.0, dtype=dtype, device=device)
    t = base[first:].view(rows, cols + pad)[:, :cols]
    t.copy_(torch.randn(rows, cols, generator=g, device=device) * scale)
    return t

def empty_like(t, value=77.0):
    """a matrix of t's shape and strides within a buffer of its own that holds `value` everywhere"""
    base = torch.full((t._base.numel() if t._base is not None else t.numel(),), value, dtype=t.dtype, device=t.device)
    return base.as_strided(t.shape, t.stride(), t.storage_offset())

def untouched(t, value=77.0):
    """nothing was written around t in its buffer"""
    base = t._base if t._base is not None else t
    m = torch.ones(base.numel(), dtype=torch.bool, device=t.device)
    m.as_strided(t.shape, t.stride(), t.storage_offset()).fill_(False)
    return bool((base.reshape(-1)[m] == value).all())

def assert_within(got, want, bound, what=""):
    """|got - want| <= bound everywhere (all float64 or broadcast to it); where want is not finite got equals it"""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaNs in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities"
    over = torch.where(fine, (got - want).abs() - bound, torch.full_like(want, -1.0))
    worst = int(over.argmax()) if over.numel() else 0
    assert not over.numel() or over.max() <= 0, f"{what}: element {worst}: {got.reshape(-1)[worst].item()} against {want.reshape(-1)[worst].item()}, over its bound by {over.max().item()}"

def generator(seed, device="cuda"):
    g = torch.Generator(device=device); g.manual_seed(seed); return g
