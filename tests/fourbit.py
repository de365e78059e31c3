"""Numbers held in 4 bits, written and read by plain loops over their definition, in 64 bits."""
import numpy as np
import torch

GROUP = 32


def bf16(x):
    """float64 numbers rounded to bfloat16."""
    return torch.as_tensor(np.asarray(x)).to(torch.float32).to(torch.bfloat16).double().numpy()


def encode(x):
    """Codes, s and m of a group of numbers."""
    lo, hi = x.min(), x.max()
    s, m = bf16((hi - lo) / 15), bf16(lo)
    codes = np.clip(np.rint((x - m) / s), 0, 15) if s > 0 else 0 * x
    return codes.astype(np.int64), s, m


def words_of(s, m):
    """The 32-bit words of scales and least values."""
    return torch.stack([torch.as_tensor(np.asarray(s)), torch.as_tensor(np.asarray(m))], -1).to(torch.float32).to(torch.bfloat16).contiguous().view(torch.uint8).numpy()


def page_bytes(values, ps):
    """[pages, kv heads, slots, d] numbers -> the pages' bytes; what the padding of a head's last group holds is zero."""
    pages, nkv, _, d = values.shape
    groups = -(-d // GROUP)
    out = np.zeros((pages, nkv, ps * groups * 20), np.uint8)
    codes = out[..., :groups * ps * 16].reshape(pages, nkv, groups, ps, 16)
    words = np.zeros((pages, nkv, ps, groups, 4), np.uint8)
    for j in range(groups):
        g = values[..., j * GROUP:min(d, (j + 1) * GROUP)]
        lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
        s, m = bf16((hi - lo) / 15), bf16(lo)
        c = np.where(s > 0, np.clip(np.rint((g - m) / np.where(s > 0, s, 1)), 0, 15), 0).astype(np.uint8)
        full = np.zeros((*g.shape[:-1], GROUP), np.uint8)
        full[..., :g.shape[-1]] = c
        codes[:, :, j] = full[..., 0::2] | (full[..., 1::2] << 4)
        words[:, :, :, j] = words_of(s[..., 0], m[..., 0])
    out[..., :groups * ps * 16] = codes.reshape(pages, nkv, -1)
    out[..., groups * ps * 16:] = words.reshape(pages, nkv, -1)
    return out


def page_parts(data, ps, d):
    """Bytes of pages -> codes [pages, kv heads, slots, d], s and m [pages, kv heads, slots, groups]."""
    groups = -(-d // GROUP)
    pages, nkv, _ = data.shape
    codes = data[..., :groups * ps * 16].reshape(pages, nkv, groups, ps, 16)
    two = np.stack([codes & 15, codes >> 4], -1).reshape(pages, nkv, groups, ps, GROUP).transpose(0, 1, 3, 2, 4).reshape(pages, nkv, ps, -1)[..., :d]
    words = torch.from_numpy(np.ascontiguousarray(data[..., groups * ps * 16:])).view(torch.bfloat16).double().numpy().reshape(pages, nkv, ps, groups, 2)
    return two, words[..., 0], words[..., 1]


def page_values(data, ps, d):
    codes, s, m = page_parts(data, ps, d)
    at = np.arange(d) // GROUP
    return m[..., at] + s[..., at] * codes


def weight_values(data, group, n, k):
    """The bytes of a weight (weights.pack4) -> its values, column by column."""
    out = np.zeros((data.shape[0] * 16, data.shape[1] * 128))
    words = torch.from_numpy(np.ascontiguousarray(data[..., 1024:])).view(torch.bfloat16).double().numpy().reshape(*data.shape[:2], 16, 128 // group, 2)
    for r in range(16):
        for c in range(128):
            j, t, e = c // 32, c % 32 // 8, c % 8
            half = (e % 2) * 4 + e // 2
            byte = 512 * (r // 8) + 64 * (r % 8) + 16 * t + 4 * j + half // 2
            code = (data[..., byte] >> (4 * (half % 2))) & 15
            out[r::16, c::128] = words[:, :, r, c // group, 1] + words[:, :, r, c // group, 0] * code
    return out[:n, :k]
