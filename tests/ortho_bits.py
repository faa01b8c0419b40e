"""How many bits an orthogonalisation may lose (shared by the CPU and the GPU
tests of it): the bound, the definition in float64, the plain float32 form, and
a CPU model of the tensor-core path's arithmetic in which single terms of its
products can be left out."""
import math

import torch

DEFAULT = ((3.4445, -4.7750, 2.0315),) * 5
SCHEDULES = {"default": DEFAULT, "two": ((3.0, -4.0, 1.75), (2.0, -1.5, 0.5))}
PRODUCTS = ("gram", "poly", "apply")


def definition(U, coefs):
    """One matrix, float64."""
    X = U.double()
    X = X / X.norm()
    tall = X.shape[0] > X.shape[1]
    X = X.T if tall else X
    for a, b, c in coefs:
        A = X @ X.T
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.T if tall else X


def plain(U, coefs):
    """The same steps in float32 throughout, the norm in float64."""
    X = (U.double() / U.double().norm()).float()
    tall = X.shape[0] > X.shape[1]
    X = X.T if tall else X
    for a, b, c in coefs:
        A = X @ X.T
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.T if tall else X


def bound(ref, plain_out):
    """What |O - O64|_F may be.  The iterates carry 22 bits against float32's
    24, so every rounding is up to four times plain float32's, and what the
    steps make of it is what they make of plain float32's on the same matrix;
    2^-20 of the result besides, for the roundings that the float32 form does
    not have (the products' dropped low-by-low terms, the split of the matrix)
    and for a float32 run that happens to be lucky."""
    return 4.0 * float((plain_out.double() - ref).norm()) + 2.0**-20 * float(ref.norm())


def small_entries_bound(m, coefs):
    """What the planes' fixed step adds to the error of one column of O (its
    2-norm, m rows).  X is held before step k in units of which its bound x_max
    is more than 2^14, with an error of at most 2^-25 where the low plane is
    subnormal: 2^-39 x_max an entry; the steps from k on multiply it by at most
    the product of their b_max."""
    total, rest = 0.0, 1.0
    for _, _, _, x_max, b_max in reversed(plan(coefs)):
        rest *= b_max
        total += x_max * rest
    return math.sqrt(m) * 2.0**-39 * total


# ---- the tensor-core path's arithmetic ----------------------------------------


def _scale_for(most):
    return 2.0 ** (15.0 - math.ceil(math.log2(max(most, 1e-3))))


def plan(coefs):
    """Per step (a, b, c, largest singular value before it, largest |a + bs + cs^2|)."""
    out, top = [], 1.0
    for a, b, c in coefs:
        s = torch.linspace(0.0, top * top, 100001, dtype=torch.float64)
        f = (a + s * (b + s * c)).abs()
        out.append((a, b, c, top, float(f.max())))
        top = max(1e-3, float((s.sqrt() * f).max()) * 1.01)
    return out


def _planes(v):
    v = v.float()
    hi = v.half()
    return hi.double(), (v - hi.float()).half().double()


def _product(left, right, drop):
    out = left[0] @ right[0]
    if drop != "left":
        out = out + left[1] @ right[0]
    if drop != "right":
        out = out + left[0] @ right[1]
    return out.float().double()


def model(U, coefs, drop=None):
    """The path's arithmetic; ``drop``: (product, "left" or "right"), whose low
    plane that product leaves out."""
    def dropped(product):
        return drop[1] if drop is not None and drop[0] == product else None

    steps = plan(coefs)
    sx = _scale_for(steps[0][3])
    V = U.float()
    tall = V.shape[0] > V.shape[1]
    V = V.T if tall else V
    X = _planes(V * torch.tensor(sx / float(U.double().norm()), dtype=torch.float32))
    eye = torch.eye(V.shape[0], dtype=torch.float64)
    for k, (a, b, c, x_max, b_max) in enumerate(steps):
        sa, sb, sc = _scale_for(x_max * x_max), _scale_for(b_max), _scale_for(abs(b) + abs(c) * x_max * x_max)
        A = (_product(X, (X[0].T, X[1].T), dropped("gram")) * (sa / (sx * sx))).float().double()
        C = (A * (c * sc / sa) + eye * (b * sc)).float()
        B = (_product(_planes(A), _planes(C), dropped("poly")) * (sb / (sa * sc)) + eye * (a * sb)).float()
        Y = _product(_planes(B), X, dropped("apply"))
        if k + 1 == len(steps):
            out = (Y / (sb * sx)).float()
            return out.T if tall else out
        sn = _scale_for(steps[k + 1][3])
        X, sx = _planes(Y * (sn / (sb * sx))), sn
