"""The distillation loss of include/credit.h, term by term over dense rows in 64
bits: differentiable in the logits, written apart from the oracle."""
import torch


def dense_q(ids: torch.Tensor, teacher: torch.Tensor, cols: int, tail: bool,
            temperature: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(q [cols], which columns an entry names) of one row: entries that name one
    column add up."""
    live = ids >= 0
    t = teacher[live].double()
    q = t.exp() if tail else torch.softmax(t / temperature, dim=0)
    named = torch.zeros(cols, dtype=torch.bool)
    named[ids[live]] = True
    return torch.zeros(cols, dtype=torch.float64).index_add_(0, ids[live], q), named


def loss(z: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, tail: bool,
         temperature: float = 1.0) -> torch.Tensor:
    """KL a row: sum over columns of q (ln q - ln p), with the tail's term where
    the columns outside the entries have mass."""
    rows = []
    for x, i, t in zip(z.double(), ids, teacher):
        if not (i >= 0).any():
            rows.append(x.new_zeros(()))
            continue
        q, named = dense_q(i, t, len(x), tail, temperature)
        lp = torch.log_softmax(x / temperature, dim=0)
        used = named & (q > 0)
        kl = (q[used] * (q[used].log() - lp[used])).sum()
        others = ~named & (x.detach() != -torch.inf)
        rest = (1.0 - q.sum()).clamp(min=0.0)
        if tail and others.any() and rest > 0:
            kl = kl + rest * (rest.log() - lp[others].logsumexp(0))
        rows.append(kl)
    return torch.stack(rows)


def gradient(z: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, dloss: torch.Tensor,
             tail: bool, temperature: float = 1.0) -> torch.Tensor:
    x = z.detach().double().clone().requires_grad_()
    (loss(x, ids, teacher, tail, temperature) * dloss.double()).sum().backward()
    return x.grad
