"""Which tiles and cuts linear's products take by the rule in linear.hip, from that file's own tables: for tests that have to reach every kernel."""
import math
import os
import re

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256


def kinds(bits):
    """The rule's table: (rows, columns, inner indices of a stage, two share a CU, times)."""
    with open(os.path.join(_ROOT, "allan-poe_amd", "csrc", "linear.hip")) as f:
        body = re.search(r"LIN_KINDS%s\[\] = \{(.*?)\};" % ("" if bits == 16 else "_FLOAT"), f.read(), re.S).group(1)
    rows = re.findall(r"\{([^{}]*)\}", body)
    return [tuple({"true": 1.0, "false": 0.0}[v] if v in ("true", "false") else float(v.rstrip("f")) for v in (c.strip() for c in r.split(","))) for r in rows]


def choose(m, n, k, bits, parts=1, cus=CUS, time=False):
    """(kind, whether the inner side is cut) of an m x n product over k; with `time` what the rule says it takes, in us."""
    best, least = None, math.inf
    for number, (bm, bn, ke, two, fixed, inner, alone_fixed, alone_inner) in enumerate(kinds(bits)):
        tiles, stages = -(-m // int(bm)) * -(-n // int(bn)), -(-k // int(ke))
        cuts = 1
        while cuts <= 16 and (cuts == 1 or (stages // cuts >= 4 and tiles * cuts <= 2 * cus)):
            each = max(1, -(-stages // cuts))
            groups, length = tiles * cuts, each * ke * parts
            rounds = -(-groups // (2 * cus if two else cus))
            t = 3 + rounds * (alone_fixed + alone_inner * length if two and groups <= cus else fixed + inner * length)
            t += 3 + (cuts + 1) * m * n * 1e-6 if cuts > 1 else 0
            if t < least:
                best, least = (number, -(-stages // each) > 1), t
            cuts += 1
    return least if time else best


def launches(m, n, k, bits, parts=1):
    """What a call and its gradient launch: the forward product, and grad_x and grad_w in one launch or two, each with its kind, and whether it is cut."""
    x, w = choose(m, k, n, bits, parts), choose(n, k, m, bits, parts)
    out = {("forward", *choose(m, n, k, bits))} if parts == 1 else set()
    if x[0] == w[0]:
        return out | {("both", parts, x[0]), ("both, grad_x", parts, *x), ("both, grad_w", parts, *w)}
    return out | {("grad_x", parts, *x), ("grad_w", parts, *w)}


def a_float_a_load(m, n, k):
    """Whether floats that begin anywhere are read one by one in the forward product (else they are laid out anew first)."""
    return 0.15 * choose(m, n, k, 32, time=True) < 5 + (m + n) * k * 8 / 4e6
