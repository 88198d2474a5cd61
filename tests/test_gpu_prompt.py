"""attn_prompt against softmax attention in 64 bits."""
import pytest
import torch

from airframe_amd import TsError
from airframe_amd.prompt import attn_prompt, attn_prompt_workspace
from tests.packed_util import DTYPES, attend, offsets, rand

pytestmark = pytest.mark.gpu
NAMES = sorted(DTYPES)


def plain(q, k, v, off, softcap=0.0):
    """The attention of every sequence in 64 bits, on the CPU; other rows 0."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    g = q.shape[1] // k.shape[1]
    for a, b in zip(off[:-1], off[1:]):
        hidden = torch.ones(b - a, b - a, dtype=torch.bool).triu(1)
        for h in range(q.shape[1]):
            out[a:b, h] = attend(q[a:b, h], k[a:b, h // g], v[a:b, h // g], hidden, softcap)
    return out


def near(got, want, q, k, v, softcap=0.0):
    """How far an output may be off, from the roundings that the operator makes.

    With |v| <= V and scores that are off by at most D (absolute), every weight is off by a factor
    within exp(2 D), so the output moves by at most 2 V (exp(2 D) - 1).  D: the dot of head_dim
    products accumulated in f32, n 2^-24 sum |q k| / sqrt(hd) <= n 2^-24 Q K sqrt(hd) in the worst
    order (Q, K the largest elements; the typical error is far below), plus 2^-20 for exp2 and the f32 scale of
    scores below 2^4; f32 factors are kept to 22 bits, 2^-21 Q K sqrt(hd) more; softcap's tanh adds 2^-22 softcap.
    Probabilities are rounded once to the type (eps / 2, relative), the weighted sum in f32 (n keys)
    adds n 2^-24 V, and the output is rounded once (eps / 2 of it)."""
    dt, hd, n = q.dtype, q.shape[2], k.shape[0]
    big = [float(x.abs().max()) for x in (q, k, v)]
    size = big[0] * big[1] * hd ** 0.5
    d = hd * 2.0 ** -24 * size + 2.0 ** -20
    eps = torch.finfo(dt).eps / 2
    if dt == torch.float32:
        d += 2.0 ** -21 * size
        p = 2.0 ** -21
    else:
        p = eps
    d += 2.0 ** -22 * softcap
    tol = big[2] * (2 * (torch.exp(torch.tensor(2 * d)).item() - 1) + 2 * p + n * 2.0 ** -24) + eps * want.abs()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))


CASES = [([1], 1, 1, 64), ([2, 1, 0, 3], 4, 2, 8), ([33], 8, 2, 128), ([127, 65, 1], 6, 2, 80), ([31, 0, 32, 97, 64], 4, 4, 64),
         ([130], 16, 2, 256), ([200, 3], 5, 1, 200), ([96, 40], 12, 4, 96), ([260], 2, 2, 136)]


@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("lens,heads,kv,hd", CASES)
@pytest.mark.parametrize("name", NAMES)
def test_prompt(gpu, name, lens, heads, kv, hd, softcap):
    dt, off = DTYPES[name], offsets(lens)
    q, k, v = rand((off[-1], heads, hd), 1, dt), rand((off[-1], kv, hd), 2, dt), rand((off[-1], kv, hd), 3, dt)
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), off, softcap=softcap).cpu()
    assert got.dtype == dt
    near(got, plain(q, k, v, off, softcap), q, k, v, softcap)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("name", NAMES)
def test_prompt_sharp(gpu, name, hd):
    """Scores of some tens, so that a few keys dominate a row and the running maximum moves."""
    dt, off = DTYPES[name], [0, 150, 411]
    q, k, v = rand((411, 4, hd), 1, dt, 3.0), rand((411, 2, hd), 2, dt, 3.0), rand((411, 2, hd), 3, dt)
    k[::37] *= 2
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), off).cpu()
    near(got, plain(q, k, v, off), q, k, v)


@pytest.mark.parametrize("name", NAMES)
def test_prompt_magnitudes(gpu, name):
    """Values and keys of very different sizes, rows of zeros, constant rows: an output that one small
    value row dominates keeps its relative accuracy."""
    dt, n, hd = DTYPES[name], 90, 64
    q, k, v = rand((n, 2, hd), 1, dt), rand((n, 1, hd), 2, dt), rand((n, 1, hd), 3, dt)
    k[0], v[0] = 0.0, 0.0
    k[1] = k[1] * 1e-3
    v[5] = 1.0
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), [0, n]).cpu()
    near(got, plain(q, k, v, [0, n]), q, k, v)
    # one scale for all of v: the output scales with it (a power of two; in f16's range for f16)
    s = 2.0 ** (-9 if dt == torch.float16 else -40)
    small = attn_prompt(q.cuda(), k.cuda(), (v * s).cuda(), [0, n]).cpu()
    want = plain(q, k, v * s, [0, n])
    # (an f16 element of v s or of the output below 2^-14 is held to 2^-25)
    tiny = 2.0 ** -24 if dt == torch.float16 else 0.0
    assert ((small.double() - want).abs() <= tiny + (2.0 ** -6 if dt != torch.float32 else 2.0 ** -17) * float((v * s).abs().max())).all()
    # the first token attends to itself alone: its output is its value, to the type's last bit
    v[0] = rand((1, hd), 9, dt)
    first = attn_prompt(q.cuda(), k.cuda(), v.cuda(), [0, n])[0].cpu()
    assert ((first.double() - v[0].double()).abs() <= v[0].double().abs() * 2.0 ** -20 + 2.0 ** -22 * float(v[0].abs().max())
            if dt == torch.float32 else first == v[0]).all()


@pytest.mark.parametrize("hd", [64, 256])
def test_prompt_f32_value_ranges(gpu, hd):
    """f32 value rows from 1e-25 to 1e30 next to each other: every row's output is within the bound of its
    own largest value that it sees (2^-18: 22 bits of every factor, and scores of some units)."""
    n = 130
    q, k, v = rand((n, 2, hd), 1), rand((n, 1, hd), 2), rand((n, 1, hd), 3)
    v *= torch.tensor([10.0 ** (-25 + 55 * ((7 * i) % n) / (n - 1)) for i in range(n)])[:, None, None]
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), [0, n]).cpu().double()
    want = plain(q, k, v, [0, n])
    seen = v.abs().amax((1, 2)).cummax(0).values.double()[:, None, None]
    assert ((got - want).abs() <= 2.0 ** -18 * seen).all()


@pytest.mark.parametrize("scale", [1e-20, 1e25])
def test_prompt_f32_small_and_large(gpu, scale):
    """All values tiny or huge: the relative accuracy stays."""
    n, hd = 70, 128
    q, k, v = rand((n, 4, hd), 1), rand((n, 2, hd), 2), rand((n, 2, hd), 3)
    want = attn_prompt(q.cuda(), k.cuda(), v.cuda(), [0, n]).cpu().double()
    got = attn_prompt(q.cuda(), k.cuda(), (v * scale).cuda(), [0, n]).cpu().double() / scale
    assert ((got - want).abs() <= 2.0 ** -20 * 5).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("name", NAMES)
def test_prompt_masked_values(gpu, name, hd):
    """Infinities and NaN at tokens that a row does not see leave it as it was, bit for bit; rows that
    see them get what the sum gives."""
    dt, n = DTYPES[name], 140
    q, k, v = (x.cuda() for x in (rand((n, 4, hd), 1, dt), rand((n, 2, hd), 2, dt), rand((n, 2, hd), 3, dt)))
    off = [0, 100, n]
    want = attn_prompt(q, k, v, off)
    for at in (3, 50, 99):
        for what in (float("inf"), float("-inf"), float("nan")):
            k2, v2 = k.clone(), v.clone()
            v2[at, 0, 5] = what
            v2[at, 1, hd - 1] = what
            got = attn_prompt(q, k, v2, off)
            assert torch.equal(got[:at], want[:at]) and torch.equal(got[100:], want[100:])
            seen = got[at:100]
            for d, heads in ((5, slice(0, 2)), (hd - 1, slice(2, 4))):
                hit = seen[:, heads, d].float()
                assert hit.isnan().all() if what != what else (hit == what).all()
            clean = [d for d in range(hd) if d != 5]
            # (the finite dims of a row that sees one: f32's value row with an infinity is held in f16 alone)
            tol = 2.0 ** -9 if dt == torch.float32 else 0.0
            assert ((seen[:, 0][:, clean].float() - want[at:100, 0][:, clean].float()).abs() <= tol).all()
            k2[at, 0, 1] = what
            got = attn_prompt(q, k2, v, off)
            assert torch.equal(got[:at], want[:at]) and torch.equal(got[100:], want[100:])
            assert torch.equal(got[:, 2:], want[:, 2:])


@pytest.mark.parametrize("name", NAMES)
def test_prompt_strided_rows(gpu, name):
    """q, k and v as parts of one fused row, the output into a wider one; rows outside the offsets
    are neither read nor written."""
    dt, hd = DTYPES[name], 64
    wide = rand((75, 8, hd), 1, dt).cuda()
    wide[:3], wide[70:] = float("nan"), float("nan")
    off = [3, 3, 41, 70]
    out = torch.full((80, 6, hd), 5.0, dtype=dt, device="cuda")
    attn_prompt(wide[:, :4], wide[:, 4:6], wide[:, 6:], off, out=out[:, 1:5])
    q, k, v = (wide[3:70, a:b].contiguous() for a, b in ((0, 4), (4, 6), (6, 8)))
    want = attn_prompt(q, k, v, [0, 38, 67])
    assert torch.equal(out[3:70, 1:5], want)
    assert (out[:3] == 5).all() and (out[70:] == 5).all() and (out[:, 0] == 5).all() and (out[:, 5] == 5).all()
    fresh = attn_prompt(wide[:, :4], wide[:, 4:6], wide[:, 6:], torch.tensor(off, dtype=torch.int32))
    assert torch.equal(fresh[3:70], want) and (fresh[:3] == 0).all() and (fresh[70:] == 0).all()


@pytest.mark.parametrize("name", NAMES)
def test_prompt_many_sequences(gpu, name):
    """Past one launch's table, lengths of 0 to 3 (a softmax over at most 3 keys)."""
    dt = DTYPES[name]
    lens = [(7 * i) % 4 for i in range(261)]
    off = offsets(lens)
    q, k, v = rand((off[-1], 3, 24), 1, dt), rand((off[-1], 1, 24), 2, dt), rand((off[-1], 1, 24), 3, dt)
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), off).cpu()
    near(got, plain(q, k, v, off), q, k, v)


@pytest.mark.parametrize("name", NAMES)
def test_prompt_long(gpu, name):
    """A long prompt next to a short one, checked at rows spread over it; the same rows twice give the
    same bits."""
    dt, n, hd = DTYPES[name], 2600, 128
    q, k, v = rand((n, 4, hd), 1, dt), rand((n, 1, hd), 2, dt), rand((n, 1, hd), 3, dt)
    off = [0, 2590, n]
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), off)
    assert torch.equal(got, attn_prompt(q.cuda(), k.cuda(), v.cuda(), off))
    got = got.cpu()
    for t in (0, 1, 63, 64, 1023, 1024, 2047, 2588, 2589, 2590, 2599):
        a = 0 if t < 2590 else 2590
        for h in range(4):
            want = attend(q[t:t + 1, h], k[a:t + 1, 0], v[a:t + 1, 0], torch.zeros(1, t + 1 - a, dtype=torch.bool))
            near(got[t:t + 1, h], want, q, k[a:t + 1], v)


def test_prompt_graph_and_stream(gpu):
    """Captured once (f32, with its scratch), replayed between eager work; and on a side stream."""
    off = [0, 70, 100]
    q, k, v = (torch.zeros(100, h, 64, device="cuda") for h in (4, 2, 2))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        attn_prompt(q, k, v, off)
        with torch.cuda.graph(graph, stream=side):
            out = attn_prompt(q, k, v, off)
    for i in range(4):
        for j, x in enumerate((q, k, v)):
            x.copy_(rand(tuple(x.shape), 10 * i + j).cuda())
        graph.replay()
        want = attn_prompt(q, k, v, off)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        got = attn_prompt(q, k, v, off, stream=side)
        side.synchronize()
        assert torch.equal(got, want)


def test_prompt_refusals(gpu):
    q, k = torch.zeros(10, 4, 64).cuda(), torch.zeros(10, 2, 64).cuda()
    assert attn_prompt(q[:0], k[:0], k[:0], [0, 0]).shape == (0, 4, 64)
    for bad in (lambda: attn_prompt(q, k, k[..., :32], [0, 10]), lambda: attn_prompt(q, k.half(), k, [0, 10]),
                lambda: attn_prompt(q, k, k, [0, 11]), lambda: attn_prompt(q, k[:5], k, [0, 10]), lambda: attn_prompt(q, k, k, [0]),
                lambda: attn_prompt(q.double(), k.double(), k.double(), [0, 10]),
                lambda: attn_prompt(q, k, k, [0, 10], out=q[:5]), lambda: attn_prompt(q, k, k, [0, 10], out=q.half()),
                lambda: attn_prompt(q.cpu(), k, k, [0, 10])):
        with pytest.raises(ValueError):
            bad()
    big = torch.zeros(10, 1, 264).cuda()
    small = torch.zeros(attn_prompt_workspace(torch.float32, 9, 2, 64), dtype=torch.uint8, device="cuda")
    for bad, code in ((lambda: attn_prompt(q, k, k, [0, 6, 5]), -1), (lambda: attn_prompt(q, k, k, [-1, 5]), -1),
                      (lambda: attn_prompt(q[:, :3].contiguous(), k, k, [0, 10]), -1), (lambda: attn_prompt(q, k, k, [0, 10], out=q), -1),
                      (lambda: attn_prompt(q, k, k, [0, 10], softcap=-1.0), -1), (lambda: attn_prompt(big, big, big, [0, 10]), -3),
                      (lambda: attn_prompt(q[..., :4].contiguous(), k[..., :4].contiguous(), k[..., :4].contiguous(), [0, 10]), -1),
                      (lambda: attn_prompt(q, k, k, [0, 10], workspace=small), -6)):
        with pytest.raises(TsError) as e:
            bad()
        assert e.value.code == code
