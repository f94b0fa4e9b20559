"""Error bounds of the row operators' single-precision sums, term by term, for the tests that need them tighter than one
constant for all sizes.

A term 2^d of a row's softmax: ex2 is good to 2^-22. Its exponent d = x*kappa - shift, or (x - max)*kappa, carries at most
three roundings of 2^-24 |d| (kappa's, the product's or the sum's, and in the second form the difference's). In a row's sum
they are weighed by the terms: sum p |d| <= log2 V + 2. A lane adds its terms one after the other, 2^-24 of the sum each,
and raises its sum to a new maximum at most once for four vectors (16 elements and more): ex2 and two roundings, six 2^-24
for 16 additions. Lanes and warps are joined in at most 9 + 16 additions, behind one more raise each; the rounding of the
shift is undone by one more ex2. Together (1.5 terms a lane + 2.1 (log2 V + 2) + 48) 2^-24."""
import math


def terms_a_lane(V, size):
    """Most terms that a lane adds up: rows in registers have at most 64 a lane, a warp's long rows 2048 vectors in its 32
    lanes, a CTA's rows a 256th, to whole steps of four vectors."""
    per = 16 // size
    vectors = (V + 2 * per - 2) // per
    if vectors <= 256:
        return 64
    return max(math.ceil(vectors / 32 / 4) * 4 * per if vectors <= 2048 else 0, math.ceil(vectors / 256 / 4) * 4 * per)


def sum_error(V, size):
    """Relative error of a row's sum; double's is what its 2^-53 leave of the same count."""
    unit = 2.0 ** -53 if size == 8 else 2.0 ** -24
    return (1.5 * terms_a_lane(V, size) + 2.1 * (math.log2(V) + 2) + 48) * unit


def term_error(size):
    """Relative error of one term that is not flushed: |d| < 126 (1100 in double), three roundings of it and ex2's."""
    return (2.1 * 1100 + 8) * 2.0 ** -53 if size == 8 else (2.1 * 126 + 8) * 2.0 ** -24
