"""The 8-bit key / value pool restated in 64 bits: places of the codes, exponents, rounding."""
import torch

PAGE, D, FLOOR = 16, 128, -96


def places(dev="cuda"):
    """Byte of token t, dimension d in a page and head: (keys, values), each [16, 128]."""
    t, d = torch.arange(PAGE, device=dev)[:, None], torch.arange(D, device=dev)
    keys = d // 64 * 1024 + t * 64 + d % 64
    values = 2048 + d // 4 * 64 + t % 8 // 2 * 16 + d % 4 * 4 + t // 8 * 2 + t % 2
    return keys, values


def decode(codes):
    """e4m3 codes (uint8) as float64."""
    return codes.view(torch.float8_e4m3fn).double()


def pool_values(kv8, scales, kind):
    """Keys (kind 0) or values (1) of a pool [pages, Hkv, 16, 128], float64."""
    return decode(kv8[:, :, places(kv8.device)[kind]].contiguous()) * torch.exp2(scales[:, :, kind, None, None].double() - 127)


def exponent(amax):
    """Smallest e >= -96 with amax <= 448 * 2^e, elementwise (float64)."""
    e = torch.where(amax > 0, torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448)), float(FLOOR))
    e = torch.where(amax > 448 * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= 448 * torch.exp2(e - 1), e - 1, e)
    return e.clamp(min=FLOOR)


def e4m3(x):
    """x (|x| <= 448) at the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def quantise(x):
    """What the pool holds of page values x [..., 16, 128]: (values, exponents); NaN and infinities become NaN."""
    fine = torch.isfinite(x)
    e = exponent(torch.where(fine, x, 0.0).abs().amax((-2, -1)))
    s = torch.exp2(e)[..., None, None]
    return torch.where(fine, e4m3(torch.where(fine, x, 0.0) / s) * s, float("nan")), e


def fill(kv8, scales, pages, kind, x):
    """Stores page values x [n, Hkv, 16, 128] of `kind` in the physical pages (exactly representable ones)."""
    v, e = quantise(x.double())
    codes = (v / torch.exp2(e)[..., None, None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    at = places(kv8.device)[kind]
    kv8[pages[:, None, None, None], torch.arange(kv8.shape[1], device=kv8.device)[:, None, None], at] = codes
    scales[pages, :, kind] = (e + 127).to(torch.uint8)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def page_table(lens, gen, extra=3, width=None):
    """Random pages for contexts `lens`: (table [B, width] on the GPU, number of pages). Unused columns hold -1."""
    need = [-(-n // PAGE) for n in lens]
    total = sum(need) + extra
    ids = torch.randperm(total, generator=gen, device="cuda").tolist()
    width = width or max(1, max(need))
    rows = []
    for n in need:
        rows.append([ids.pop() for _ in range(n)] + [-1] * (width - n))
    return ints(rows), total
