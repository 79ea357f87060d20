"""Shared pieces of the sequence operators' tests."""

import torch

# the rounding of a stored value: half a step
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Half the smallest step of the stored type (its subnormals).  fp32, which all is computed in: an
# operation whose result is below 2^-126 adds up to 2^-150, later factors (below 16) multiply
# it, and an output comes from at most 64 such operations: 64 * 16 * 2^-150 = 2^-140.
FLOOR = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def within(got, ref, err, what, dtype=None):
    """|got - ref| <= err + the rounding of the stored type, element by element."""
    dtype = dtype or got.dtype
    got, ref, err = got.detach().double().cpu(), ref.detach().double().cpu(), err.detach().double().cpu()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(ref.shape)}"
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), f"{what}: finite in other places"
    tol = err + HALF[dtype] * (ref.abs() + err) + FLOOR[dtype]
    ok = ((got - ref).abs() <= tol) | ~torch.isfinite(ref)
    if not bool(ok.all()):
        i = ((got - ref).abs() / tol).nan_to_num().argmax()
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} outside; worst {got.flatten()[i]:.9g} "
                             f"for {ref.flatten()[i]:.9g}, allowed {tol.flatten()[i]:.3g}")
