"""cq_attention where finite scales differ by many powers of two between keys: what a token does not see, or gives no weight, does not take bits from what it
does see.

Bounds are those of attention_reference.py for the entries that a token gives weight to, and what 16 bits below the largest scale may lose on the matrix cores.
Where scales differ by up to 2^12: of a weight, half of f16's smallest step, 2^-25, of a largest weight of at least 2^5, times 2^12, so 2^-18 |v_j| of each key; of an entry
that is made a number of f16, 2^-25 of numbers up to 2 (2^12 times its scale), so 2^-12 of its scale, of a key's entry times |q| in the score.  Where they differ by more, tokens stay there
whose results are 2^15 times what they may have lost, so 2^-15 of the largest of 16 or 32 neighbouring entries, and whose scores are off by 2^-12 (times ln 2) at most."""
import numpy as np
import pytest

from attention_reference import Attention
from cubek_amd import ElemType, QuantStore, QuantValue
from matmul_reference import check_rounded, scheme_of

pytestmark = pytest.mark.gpu
F16, BF16 = ElemType.F16, ElemType.BF16
U32, NATIVE = QuantStore.U32, QuantStore.Native
V = QuantValue
CODES = {"q8": (V.Q8S, NATIVE), "q8_words": (V.Q8F, U32), "q4": (V.Q4S, U32), "e4m3": (V.E4M3, NATIVE), "e5m2": (V.E5M2, NATIVE), "e2m1": (V.E2M1, NATIVE), "ocp": (V.E2M1_OCP, U32)}
FACTORS = [2.0 ** 10, 2.0 ** 13, 2.0 ** 20, 2.0 ** 40, 2.0 ** 100]


def scheme(name, block, param=0):
    return scheme_of(CODES[name][0], [block], param, CODES[name][1])


def far_bound(want, size):
    """What is added to a bound for scales that differ by more than 2^12."""
    tiles = np.abs(want).reshape(want.shape[:2] + (-1, 32)).max(-1).repeat(32, -1)
    return 2.0 ** -15 * tiles + 2.0 * size * 2.0 ** -12 * np.log(2.0)


def spread_bound(case, size, scale):
    """The same for those that differ by less."""
    of = [float(pool.scales.double().abs().max()) for pool in (case.k, case.v)]
    extra = np.zeros(case.q.shape)
    q = case.q.double().abs().sum(-1).numpy()[..., None]
    for s, (n, _) in enumerate(case.sequences):
        a = case.offsets[s]
        for head in range(case.q.shape[1]):
            extra[a:a + n, head] = 2.0 ** -18 * np.abs(case.of_sequence(case.v, s, head // case.group)).sum(0)
    return extra + 2.0 ** -12 * of[1] + 2.0 * size * scale * q * 2.0 ** -12 * of[0]


def sizes(case, **scores):
    """sum_j p_j |v_j|"""
    held, case.v.entries = case.v.entries, np.abs(case.v.entries)
    size, _ = case.want(**scores)
    case.v.entries = held
    return size


class enlarged:
    """The scales of a key `factor` times what they are, for a while."""

    def __init__(self, case, of, s, keys, factor):
        page = case.k.entries.shape[2]
        self.pool, self.factor = case.v if of == "v" else case.k, factor
        self.at = (case.table[s, np.asarray(keys) // page], slice(None), np.asarray(keys) % page)

    def __enter__(self):
        self.kept = self.pool.scales[self.at].clone(), self.pool.entries[self.at].copy()
        self.pool.scales[self.at] = self.kept[0] * self.factor
        self.pool.entries[self.at] = self.kept[1] * self.factor

    def __exit__(self, *_):
        self.pool.scales[self.at], self.pool.entries[self.at] = self.kept


SHAPES = [(64, 32), (128, 128), (256, 32), (128, 32), (64, 64), (192, 64), (256, 64)]
OF_CODE = {name: [SHAPES[i], SHAPES[(i + 1) % 7], SHAPES[(i + 3) % 7]] for i, name in enumerate(CODES)}


@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("tokens", [5, 20, 150])
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_large_scales_of_a_last_token(oracle, name, tokens, elem):
    """The last token alone sees them: of keys, of values, in the step of the others and in a later one."""
    for dim, block in OF_CODE[name]:
        for seed, length in enumerate((tokens, 23 * 32 + tokens)):
            case = Attention(oracle, seed, [(tokens, length), (tokens, tokens + 3)], 4, 2, dim, 16, elem, scheme(name, block))
            want, bound = case.want()
            size = sizes(case)
            bound = bound + far_bound(want, size) + spread_bound(case, size, dim ** -0.5)
            rows = np.arange(case.tokens) != tokens - 1
            for of, factor in [("v", f) for f in FACTORS] + [("k", f) for f in FACTORS[1:]]:
                with enlarged(case, of, 0, [length - 1], factor):
                    got = case.call().double().cpu().numpy()
                    check_rounded(got[rows], want[rows], bound[rows], elem, (dim, of, factor, length))
                    if of == "v" and elem == BF16 and factor == FACTORS[-1]:  # the token that sees it: f32's range, and bf16's
                        its, its_bound = case.want()
                        check_rounded(got[~rows], its[~rows], its_bound[~rows], elem, ("the last", dim, length))


@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("tokens", [3, 20, 150])
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_large_scales_behind_a_window(oracle, name, tokens, elem):
    """The first token alone sees them, for the others' windows have passed."""
    for dim, block in OF_CODE[name][:2]:
        case = Attention(oracle, 2, [(tokens, 700), (tokens, tokens + 3)], 4, 2, dim, 16, elem, scheme(name, block, 2))
        want, bound = case.want(window=100)
        bound = bound + far_bound(want, sizes(case, window=100))
        for of in "vk":
            for factor in FACTORS[2:]:
                with enlarged(case, of, 0, [700 - tokens - 99], factor):
                    got = case.call(window=100).double().cpu().numpy()
                check_rounded(got[1:], want[1:], bound[1:], elem, (dim, of, factor))


@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("tokens", [1, 3, 20, 150])
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_large_values_without_weight(oracle, name, tokens, elem):
    """All tokens see a key with a bias that leaves it less than e^-200 of their weight: it counts as nothing, many keys back or a few, in a wave's first step or
    in that of the keys that have weight."""
    for dim, block in OF_CODE[name][:2]:
        case = Attention(oracle, 3, [(tokens, 960 + tokens), (tokens, tokens + 3)], 4, 2, dim, 16, elem, scheme(name, block))
        for back, slope in ((900, 0.5), (20, 16.0)):
            slopes = np.full(4, slope, np.float32)
            want, bound = case.want(slopes=slopes)
            bound = bound + far_bound(want, sizes(case, slopes=slopes))
            for factor in FACTORS[2:]:
                for workspace in (True, False):
                    with enlarged(case, "v", 0, [959 - back], factor):
                        got = case.call(workspace, slopes=slopes).double().cpu().numpy()
                    check_rounded(got, want, bound, elem, (dim, back, factor, workspace))


@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("tokens", [1, 20, 150])
@pytest.mark.parametrize("elem", [BF16, F16], ids=lambda e: e.name)
def test_small_scales_among_others(oracle, name, tokens, elem):
    """A key or a value whose scales are zero, or smaller than the others' by many powers of two, is one like any other."""
    for dim, block in OF_CODE[name][:1]:
        case = Attention(oracle, 4, [(tokens, 300), (tokens, tokens + 3)], 4, 2, dim, 16, elem, scheme(name, block))
        for of, factor in (("v", 0.0), ("v", 2.0 ** -30), ("k", 2.0 ** -30), ("k", 0.0)):
            with enlarged(case, of, 0, [0, 70, 299], factor):
                case.check((dim, of, factor))


@pytest.mark.parametrize("name", ["q8", "q4", "e4m3"])
@pytest.mark.parametrize("tokens", [1, 20, 150])
def test_blocks_of_entries_of_unlike_sizes(oracle, name, tokens):
    """The same blocks of every value are 2^-24 times as large as the others: their entries keep their bits."""
    case = Attention(oracle, 5, [(tokens, 300), (tokens, tokens + 3)], 4, 2, 128, 16, BF16, scheme(name, 32))
    small = slice(32, 96)
    case.v.scales[..., 1:3] *= 2.0 ** -24
    case.v.entries[..., small] *= 2.0 ** -24
    got = case.call().double().cpu().numpy()
    want, bound = case.want()
    check_rounded(got, want, bound, BF16, "all")
    case.v.entries[..., :32] = case.v.entries[..., 96:] = 0.0  # nothing of a bound of the small ones goes by the large ones
    want, bound = case.want()
    check_rounded(got[..., small], want[..., small], bound[..., small], BF16, "small")
