"""Plain forms, in 64 bits, of keys and values held in 4 bits and of attention over them."""

import math

import torch

GROUP = 64


def quantize4(x):
    """What a cache of 4 bits holds for heads [..., hd], as float64 values."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a in range(0, x.shape[-1], GROUP):
        part = x[..., a:a + GROUP].double().nan_to_num(nan=0.0).clamp(-3.4028234663852886e38,
                                                                      3.4028234663852886e38)
        lo = part.amin(-1, keepdim=True).clamp(max=0)
        hi = part.amax(-1, keepdim=True).clamp(min=0)
        # the step is a held number: float32's difference and quotient, then float16
        fifteen = torch.full((), 15.0, device=x.device)
        step = ((hi.float() - lo.float()) / fifteen).clamp(max=65504.0).half().double()
        by = torch.where(step > 0, step, torch.ones_like(step))
        zero = (-lo / by).round().clamp(max=15)
        out[..., a:a + GROUP] = step * (((part / by).round() + zero).clamp(0, 15) - zero)
    return out


def attention(q, k_of, v_of, batch, *, num_kv_heads, scale, window=None, sink=None, chunk=None,
              softcap=None, slopes=None, q_temp=None, keep_first=0):
    """(outputs [T, nq, hd], the same of the values' magnitudes) in float64; `k_of[e]`, `v_of[e]`:
    the entry's keys and values [context, nkv, hd] by position."""
    nq = q.shape[1]
    group = nq // num_kv_heads
    out, size = (torch.empty(q.shape, dtype=torch.float64) for _ in range(2))
    entries, positions = batch.entry_of_token.tolist(), batch.positions.tolist()
    q = q.double().cpu()
    for t, (e, p) in enumerate(zip(entries, positions)):
        lo = 0 if window is None else max(0, p - window + 1)
        if chunk is not None:
            lo = max(lo, p // chunk * chunk)
        keys = torch.cat([torch.arange(min(keep_first, lo)), torch.arange(lo, p + 1)])
        temp = 1.0 if q_temp is None else 1.0 + q_temp[0] * math.log((p + 1) // q_temp[1] + 1)
        k, v = k_of[e][keys], v_of[e][keys]
        for h in range(nq):
            s = k[:, h // group] @ q[t, h] * (scale * temp)
            if softcap is not None:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * (p - keys).double()
            if sink is not None:
                s = torch.cat([s, sink[h:h + 1].double().cpu()])
            w = torch.softmax(s, 0)[:len(keys)]
            out[t, h], size[t, h] = w @ v[:, h // group], w @ v[:, h // group].abs()
    return out, size
