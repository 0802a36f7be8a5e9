"""Plain statements of the serving operators: packed 4-bit products and attention in 64 bits,
the 8-bit block cache's append in the 32-bit steps its codes are defined by, the block
planning in Python integers.  Test infrastructure; everything on the CPU.

Besides its result each product returns the sum of magnitudes its rounding errors scale with.
"""
import torch

CODE_HALF = {torch.float8_e4m3fn: 448.0, torch.int8: 127.5}
EPS = torch.finfo(torch.float32).eps


def unpack4(words, count, dim=1):
    """codes 0 ... 15 of int32 words along `dim`, the first `count` of them"""
    shifts = torch.arange(0, 32, 4)
    codes = (words.long().unsqueeze(-1) >> shifts) & 15
    if dim == 1:
        return codes.flatten(1)[:, :count]
    return codes.permute(0, 2, 1).flatten(0, 1)[:count]


def pack4(codes, dim=1):
    """inverse of unpack4: [n, k] integers 0 ... 15"""
    if dim == 0:
        return pack4(codes.t(), 1).t().contiguous()
    n, k = codes.shape
    padded = torch.zeros(n, -(-k // 8) * 8, dtype=torch.long)
    padded[:, :k] = codes
    word = (padded.view(n, -1, 8) << torch.arange(0, 32, 4)).sum(-1)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)


def packed_linear(x, packed, scale, zero=None, bias=None):
    """-> (y, magnitudes) in float64"""
    n, k, groups = packed.shape[0], x.shape[1], scale.shape[1]
    u = unpack4(packed, k).double().view(n, groups, k // groups)
    z = torch.full((n, groups), 8.0, dtype=torch.float64) if zero is None else unpack4(zero, n, 0).double()
    w = ((u - z.unsqueeze(-1)) * scale.double().unsqueeze(-1)).view(n, k)
    # a kernel may sum the codes as they are stored and take the zero points off the sums
    big = ((u + z.unsqueeze(-1)) * scale.double().abs().unsqueeze(-1)).view(n, k)
    y, mag = x.double() @ w.t(), x.double().abs() @ big.t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag


def _encode(v, dtype):
    if dtype is torch.int8:
        return torch.nan_to_num(v.clamp(-128.0, 127.0).round(), nan=0.0).to(torch.int8)
    return v.clamp(-448.0, 448.0).to(dtype)


def kv_append(key, value, blocks, slots, dynamic=True):
    """updates `blocks` (key, value, key_scale, value_scale) in place, block by block"""
    k_codes, v_codes, k_scale, v_scale = blocks
    size, pool = k_codes.shape[2], k_codes.shape[0] * k_codes.shape[2]
    slots = slots.tolist()
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < pool:
            t += 1
            continue
        end = t + 1
        while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % size:
            end += 1
        block, at = slots[t] // size, slots[t] % size
        for x, codes, scale in ((key, k_codes, k_scale), (value, v_codes.transpose(2, 3), v_scale)):
            rows = x[t:end].float()
            if dynamic:
                finite = torch.where(rows.isfinite(), rows.abs(), torch.zeros_like(rows))
                fits = (finite.amax(dim=(0, 2)) / torch.tensor(CODE_HALF[codes.dtype])).clamp(min=EPS)
                old = scale[block].clone()
                scale[block] = fits if at == 0 else torch.maximum(old, fits)
                ratio = (old / scale[block]).view(-1, 1, 1)
                for h in range(codes.shape[1]):
                    if at and scale[block, h] != old[h]:
                        again = _encode(codes[block, h, :at].float() * ratio[h], codes.dtype)
                        codes[block, h, :at] = again
            new = _encode(rows / scale[block].view(1, -1, 1), codes.dtype)
            codes[block, :, at:at + end - t] = new.transpose(0, 1)
        t = end


def kv_attend(q, blocks, table, lens, starts=None, softmax_scale=None, out=None):
    """-> (out, sum of p |v|, largest sum of |q||k| of a row's scores times the scale), float64;
    rows outside every request are `out`'s"""
    k_codes, v_codes, k_scale, v_scale = blocks
    n_blocks, kv_heads, size, dim = k_codes.shape
    tokens, heads, _ = q.shape
    share = heads // kv_heads
    softmax_scale = dim ** -0.5 if softmax_scale is None else softmax_scale
    o = torch.zeros(tokens, heads, dim, dtype=torch.float64) if out is None else out.double().clone()
    mag, reach = torch.zeros_like(o), torch.zeros(tokens, heads, 1, dtype=torch.float64)
    k_all = k_codes.float().double() * k_scale.double()[..., None, None]
    v_all = v_codes.transpose(2, 3).float().double() * v_scale.double()[..., None, None]
    for r in range(len(lens)):
        q0, q1 = (r, r + 1) if starts is None else (int(starts[r]), int(starts[r + 1]))
        n = min(int(lens[r]), table.shape[1] * size)
        for t in range(q0, q1):
            seen = n - (q1 - q0) + (t - q0) + 1
            places = [j for j in range(max(0, seen)) if 0 <= int(table[r, j // size]) < n_blocks]
            o[t], mag[t] = 0, 0
            if not places:
                continue
            j = torch.tensor(places)
            b = table[r].long()[j // size]
            for h in range(heads):
                k, v = k_all[b, h // share, j % size], v_all[b, h // share, j % size]
                score = (k @ q[t, h].double()) * softmax_scale
                p = torch.softmax(score, 0)
                o[t, h] = p @ v
                mag[t, h] = p @ v.abs()
                reach[t, h] = ((k.abs() @ q[t, h].double().abs()) * softmax_scale).max()
    return o, mag, reach


def kv_plan(lens, new, table, free, num_free, size, total):
    """-> (lens, starts, slots, table, free, num_free, status) as lists; see ctmi_kv_plan"""
    requests, width, capacity = len(lens), len(table[0]) if table else 0, len(free)
    unchanged = lambda status: (list(lens), [0] * (requests + 1), [-1] * total, [list(r) for r in table],  # noqa: E731
                                list(free), num_free, status)
    ceil = lambda a: -(-a // size)  # noqa: E731
    if any(n < 0 or ceil(n + max(a, 0)) > width for n, a in zip(lens, new)):
        return unchanged(-1)
    if sum(a for a in new if a > 0) > total:
        return unchanged(-2)
    back = sum(ceil(n) for n, a in zip(lens, new) if a < 0)
    if not 0 <= num_free <= capacity or num_free + back > capacity:
        return unchanged(-3)
    want = sum(ceil(n + a) - ceil(n) for n, a in zip(lens, new) if a >= 0)
    if want > num_free + back:
        return unchanged(want - num_free - back)
    stack = list(free[:num_free])
    rows = [list(r) for r in table]
    for r in range(requests):
        if new[r] < 0:
            stack += rows[r][:ceil(lens[r])]
            rows[r] = [-1] * width
    starts, slots, after = [0], [], []
    for r in range(requests):
        add = max(new[r], 0)
        n = 0 if new[r] < 0 else lens[r]
        for column in range(ceil(n), ceil(n + add)):
            rows[r][column] = stack.pop()
        slots += [rows[r][p // size] * size + p % size if rows[r][p // size] >= 0 else -1 for p in range(n, n + add)]
        starts.append(starts[-1] + add)
        after.append(n + add)
    slots += [-1] * (total - len(slots))
    return after, starts, slots, rows, stack + [-1] * (capacity - len(stack)), len(stack), 0
