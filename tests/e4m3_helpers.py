"""The paged cache in 8 bits: its definition in 64 bits on the CPU, and inputs. The attention's definition and tolerances are those of
paged_helpers.py, over the values that the codes and scales stand for."""
import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def round_e4m3(y):
    """y (f64, at most 448 but for rounding) to the nearest number of the type, ties to even."""
    step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def scale_byte(top):
    """The byte of the least 2^e, e >= -127, with top <= 448 x 2^e; 0 for a row of zeros."""
    m, e = torch.frexp(top.double())  # 448 = 0.875 x 2^9
    return torch.where(top == 0, 0, (e - 9 + (m > 0.875) + 127).clamp(min=0))


def power(byte):
    return torch.where(byte == 255, float("nan"), torch.pow(torch.tensor(2.0, dtype=torch.float64), byte.double() - 127))


class Cache8:
    """As paged_helpers.Cache, in 8 bits: pages of codes with magnitudes that differ from row to row, dealt in random order. Rows that
    hold no key are NaN codes with NaN scales. dtype: the queries' type."""

    def __init__(self, g, lens, n_head_kv, hd, page, dtype, *, heads_first=False, spare=2, extra_width=1, scale_pad=0):
        self.lens, self.page, self.hd, self.n_head_kv, self.dtype = list(lens), page, hd, n_head_kv, dtype
        used = [-(-n // page) for n in lens]
        total = sum(used) + spare
        ids = torch.randperm(total, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max([1] + used) + extra_width), total + 7, dtype=torch.int32)  # unused entries are no page
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = ids[at:at + n]
            at += n
        shape = (total, n_head_kv, page, hd) if heads_first else (total, page, n_head_kv, hd)
        self.heads_first, self.scale_pad = heads_first, scale_pad
        self.k, self.v = (torch.full(shape, 0x7f, dtype=torch.uint8) for _ in range(2))
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.ks, self.vs = (torch.full((total, n_head_kv, page), 255, dtype=torch.uint8) for _ in range(2))
        for b, n in enumerate(lens):
            p = torch.arange(n)
            for pool, scale in ((self.k, self.ks), (self.v, self.vs)):
                x = torch.randn(n, n_head_kv, hd, generator=g) * torch.exp(0.5 * torch.randn(n, n_head_kv, 1, generator=g))
                byte = scale_byte(x.abs().amax(-1))
                y = round_e4m3(x.double() / power(byte)[..., None])
                pool[self.table[b, p // page].long(), p % page] = y.to(E4M3).view(torch.uint8)
                scale[self.table[b, p // page].long(), :, p % page] = byte.to(torch.uint8)

    def keys(self, b, n=None):
        p = torch.arange(self.lens[b] if n is None else n)
        page, row = self.table[b, p // self.page].long(), p % self.page
        return tuple((pool[page, row].contiguous().view(E4M3).double() * power(scale[page, :, row])[..., None]).to(self.dtype).double()
                     for pool, scale in ((self.k, self.ks), (self.v, self.vs)))

    def to(self, device):
        """(k, v, table, kv_len, scales) on the device."""
        def codes(t):
            t = t.transpose(1, 2).to(device).transpose(1, 2) if self.heads_first else t.to(device)
            return t.view(E4M3)

        def scales(t):
            wide = torch.full((t.shape[0], t.shape[1], t.shape[2] + self.scale_pad), 255, dtype=torch.uint8, device=device)
            wide[:, :, :t.shape[2]] = t.to(device)
            return wide.view(E8M0)[:, :, :t.shape[2]]
        return codes(self.k), codes(self.v), self.table.to(device), torch.tensor(self.lens, dtype=torch.int32, device=device), \
            [scales(self.ks), scales(self.vs)]
