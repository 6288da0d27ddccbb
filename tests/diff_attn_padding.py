"""A clip of differential attention alone and in a padded batch, its errors in units of the results' own
rounding to 16 bits."""
import torch

from tests import diff_attn_ref as R
from tests.test_gpu_diff_attn import call, operands


def errors(seed, H, Hkv, lq, lk, Lq, Lk, B, dt, causal, rows=False):
    """{name: (alone, in the batch)}: |result - exact| / |rounded exact - exact| of o, dq, dk, dv in 2-norm;
    rows: of o the largest of a row's.  The clip is the last of B that are padded to Lq, Lk, the first as
    long as that."""
    x, lam, do = operands(seed, 1, lq, H, Hkv, lk, dt)
    want = R.attention(*x, lam, do=do, dev="cuda", causal=causal)
    alone = call(x, lam, do, causal=causal)
    g = torch.Generator(device="cuda").manual_seed(seed)
    batch = []
    for t, n, L in zip((*x, do), (lq, lk, lk, lq), (Lq, Lk, Lk, Lq)):
        y = torch.randn(B, L, *t.shape[2:], device="cuda", generator=g).to(dt)
        y[1:, :n] = t
        batch.append(y)
    padded = call(batch[:3], lam, batch[3], causal=causal, q_lens=[Lq] + [lq] * (B - 1),
                  k_lens=[Lk] + [lk] * (B - 1))
    out = {}
    for n in ("o", "dq", "dk", "dv"):
        w = want[n][0]
        L = w.shape[1]
        size = (lambda t: t.flatten(2).norm(dim=2)) if rows and n == "o" else torch.Tensor.norm
        own = size(w.to(dt).double() - w)
        out[n] = tuple((size(t.double() - w) / own).max().item()
                       for t in (alone[n], padded[n][-1:, :L]))
        print("[roundings]", n, [round(v, 3) for v in out[n]], flush=True)
    return out
