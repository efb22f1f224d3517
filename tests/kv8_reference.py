"""Plain restatements of the 8-bit cache's format, its attention and the page operations, for tests (CPU, 64 bits)."""
import torch

QMAX = {"e4m3": 448.0, "int8": 127.0}


def quantise(x, fmt):
    """x (..., rows, 128) -> (codes as float64 values of the format, scale (...)): the three fp32 roundings that the
    format fixes, each of a 64-bit result."""
    y = x.double()
    amax = y.abs().amax((-1, -2))
    scale = (amax / QMAX[fmt]).float().clamp(min=2.0 ** -126)
    inv = (1.0 / scale.double()).float().double()
    z = (y * inv[..., None, None]).float().double().clamp(-QMAX[fmt], QMAX[fmt])
    if fmt == "int8":
        codes = torch.round(z)
    else:
        a = z.abs().clamp(min=2.0 ** -6)
        step = a / torch.frexp(a)[0] / 16
        codes = torch.round(z / step) * step
    bad = ~torch.isfinite(y).all(-1).all(-1)
    return torch.where(bad[..., None, None], 0.0, codes), torch.where(bad, float("nan"), scale)


def attention(q, k, v, scale):
    """q (Hq, 128), k / v (Hkv, n, 128), any types -> out (Hq, 128), logits (Hq, n), probabilities, and per output element
    the bound sum p |v| and per logit the bound sum |q| |k|, all in 64 bits."""
    hkv, n = k.shape[0], k.shape[1]
    q, k, v = q.double().view(hkv, -1, 128), k.double(), v.double()
    x = torch.matmul(q, k.transpose(1, 2)) * scale
    mass = torch.matmul(q.abs(), k.abs().transpose(1, 2)) * scale
    if n == 0:
        z = torch.zeros((q.shape[0] * q.shape[1], 128), dtype=torch.float64)
        return z, x.flatten(0, 1), x.flatten(0, 1), z, mass.flatten(0, 1)
    p = torch.softmax(x, -1)
    return (torch.matmul(p, v).reshape(-1, 128), x.reshape(-1, n), p.reshape(-1, n),
            torch.matmul(p, v.abs()).reshape(-1, 128), mass.reshape(-1, n))


def logit_error(mass):
    """How far an fp32 logit may be from the exact one: 128 products summed in fp32 in some order and two fp32
    scalings, each within 2^-24 of what it rounds."""
    return (128 + 2) * 2.0 ** -24 * mass


def output_bound(out, spread, mass, dtype):
    """Elementwise bound of an attention output: half a step of its type, the probabilities' relative error (the logits'
    errors, in the numerator and in the sum; 2^-15 for exponentials, sums and the split of a probability into two 16-bit
    parts) times sum p |v|, and the smallest number of the type."""
    dl = logit_error(mass).amax() if mass.numel() else torch.tensor(0.0)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return torch.finfo(dtype).eps / 2 * out.abs() * (1 + 2.0 ** -10) + (2 * torch.expm1(2 * dl) + 2.0 ** -15) * spread + tiny


class Pages:
    """The page operations on Python lists: lowest free page first, entries in their order, all or nothing."""

    def __init__(self, table, lens, refs, page, buffers):
        self.table, self.lens, self.refs, self.page = table.tolist(), lens.tolist(), refs.tolist(), page
        self.buffers = [b.clone() for b in buffers]
        self.width = table.shape[1]

    def _count(self, n):
        return -(-n // self.page)

    def free(self, seqs):
        bad = 0
        for s in seqs:
            if not 0 <= s < len(self.lens):
                bad += 1
                continue
            for i in range(self._count(self.lens[s])):
                self.refs[self.table[s][i]] -= 1
                self.table[s][i] = -1
            self.lens[s] = 0
        return [0, bad]

    def _free_pages(self, n):
        got = [p for p, r in enumerate(self.refs) if r == 0][:n]
        return got, n - len(got)

    def fork(self, parents, children):
        bad, todo, seen = 0, [], set()
        for p, c in zip(parents, children):
            ok = 0 <= p < len(self.lens) and 0 <= c < len(self.lens) and p != c and c not in seen and self.lens[c] == 0
            if 0 <= c < len(self.lens):
                seen.add(c)
            if ok:
                todo.append((p, c, self.lens[p]))
            else:
                bad += 1
        pages, short = self._free_pages(sum(1 for _, _, n in todo if n % self.page))
        if short:
            return [short, bad]
        for p, c, n in todo:
            full = n // self.page
            for i in range(full):
                self.table[c][i] = self.table[p][i]
                self.refs[self.table[p][i]] += 1
            if n % self.page:
                new = pages.pop(0)
                self.table[c][full] = new
                self.refs[new] = 1
                for b in self.buffers:
                    b[new] = b[self.table[p][full]]
            self.lens[c] = n
        return [0, bad]

    def extend(self, seqs, more):
        bad, todo, seen = 0, [], set()
        for s, m in zip(seqs, more):
            m = max(m, 0)
            if not 0 <= s < len(self.lens) or s in seen or self._count(self.lens[s] + m) > self.width:
                bad += 1
            else:
                todo.append((s, m))
            seen.add(s)
        pages, short = self._free_pages(sum(self._count(self.lens[s] + m) - self._count(self.lens[s]) for s, m in todo))
        if short:
            return [short, bad]
        for s, m in todo:
            for i in range(self._count(self.lens[s]), self._count(self.lens[s] + m)):
                self.table[s][i] = pages.pop(0)
                self.refs[self.table[s][i]] = 1
            self.lens[s] += m
        return [0, bad]

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        src = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(used) if self.refs[p] <= 0]
        to = list(range(len(self.refs)))
        for s, d in zip(src, dst):
            to[s] = d
            for b in self.buffers:
                b[d] = b[s]
        refs = [0] * len(self.refs)
        for p, r in enumerate(self.refs):
            if r > 0:
                refs[to[p]] = r
        self.refs = refs
        self.table = [[to[p] if p >= 0 else p for p in row] for row in self.table]
        return used
