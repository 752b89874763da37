"""Error bounds of the GPU tests that compare against 64-bit references."""
import torch

U32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of dtype's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rounded(ref, err, dtype):
    """Bound of |stored - ref| where the value before the store is within err of ref."""
    return err + half_step(dtype) * (ref.abs() + err) + tiny(dtype)


def check(got, ref, bound, what=""):
    got = got.double().to(ref.device)
    bad = ~((got - ref).abs() <= bound)
    same = (got == ref) | (got.isnan() & ref.isnan())  # infinities and NaN
    bad &= ~same
    if bad.any():
        i = bad.nonzero()[0].tolist()
        at = tuple(i)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, first at {at}: "
                             f"{got[at].item()} for {ref[at].item()} (bound {bound[at].item():.3e})")
