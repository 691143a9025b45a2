"""SiLU and GELU in doubles, right beside their own size wherever they are."""


def act_tails(y, act):
    """SiLU (act 2) or GELU's tanh form (3) of a tensor of doubles, as y sigmoid(x): (value, |x|).  No digits cancel."""
    import torch

    x = y if act == 2 else 2 * (2 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3)
    return y * torch.sigmoid(x), x.abs()
