"""Comparison with values in 64 bits, by the rounding of the type that a kernel writes."""

import torch


def assert_rounded(actual, exact, rel=0.0, absolute=0.0):
    """``actual`` is ``exact`` rounded once to its type (half a step: eps / 2 of the value, or of the smallest
    normal number below it), where ``exact`` itself may be off by ``rel`` of the value and ``absolute``."""
    info = torch.finfo(actual.dtype)
    exact = exact.double().to(actual.device)
    half = info.eps / 2
    bound = exact.abs() * (half + rel) * (1 + half) + absolute * (1 + half) + info.smallest_normal * half
    wide = actual.double()
    same = (wide == exact) | (wide.isnan() & exact.isnan())
    bad = ~(same | ((wide - exact).abs() <= bound))
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        worst = ((wide - exact).abs() / bound).masked_fill(~bad, 0).max()
        raise AssertionError(f'{int(bad.sum())} of {bad.numel()} values are off, by up to {float(worst):.3g} of the '
                             f'bound; first at {at}: {float(wide[at])} instead of {float(exact[at])}')
