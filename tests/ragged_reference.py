"""Plain forms in 64 bits of the ragged Gated-DeltaNet operators, sequence by
sequence and token by token (torch on any device)."""
import torch

BF16 = torch.bfloat16


def conv(x, w, states, cu, slots, has):
    """SiLU(conv) of every row (None where a row has no sequence) and the states after;
    the conv's sum is rounded to bf16 before SiLU, as the operator has it."""
    states, w = states.double(), w.double()
    out = torch.full(x.shape, float("nan"), dtype=torch.float64, device=x.device)
    for i, slot in enumerate(slots):
        a, z = cu[i], cu[i + 1]
        if a == z or not 0 <= slot < states.shape[0]:
            continue
        old = states[slot].T if has[i] else torch.zeros(3, x.shape[1], dtype=torch.float64, device=x.device)
        rows = torch.cat((old, x[a:z].double()))
        y = (rows.unfold(0, 4, 1) * w).sum(-1).to(BF16).double()
        out[a:z] = y * torch.sigmoid(y)
        states[slot] = rows[-3:].T
    return out, states


def normed(x):
    x = x.double()
    return x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()


def delta(q, k, v, g, beta, states, cu, slots, has, norm=normed):
    """The delta rule's rows (NaN where a row has no sequence) and the states after."""
    states = states.double()
    out = torch.full(v.shape, float("nan"), dtype=torch.float64, device=v.device)
    rep = 32 // q.shape[1]
    for i, slot in enumerate(slots):
        a, z = cu[i], cu[i + 1]
        if a == z or not 0 <= slot < states.shape[0]:
            continue
        s = states[slot] if has[i] else torch.zeros_like(states[slot])
        qn = norm(q[a:z]).repeat_interleave(rep, 1) * 128 ** -0.5
        kn = norm(k[a:z]).repeat_interleave(rep, 1)
        for t in range(z - a):
            s = s * g[a + t].double().exp()[:, None, None]
            d = (v[a + t].double() - (s * kn[t][:, :, None]).sum(1)) * beta[a + t].double()[:, None]
            s = s + kn[t][:, :, None] * d[:, None]
            out[a + t] = (s * qn[t][:, :, None]).sum(1)
        states[slot] = s
    return out, states


def cu_of(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu
