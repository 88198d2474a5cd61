"""attn_prompt against softmax attention in 64 bits, as closely as its roundings allow, and over the whole
range of scores, softcaps and sizes."""
import pytest
import torch

from airframe_amd.prompt import attn_prompt
from tests.packed_util import DTYPES, attend, attend_bound, norms, offsets, rand

pytestmark = pytest.mark.gpu
NAMES = sorted(DTYPES)


def close(q, k, v, off, softcap=0.0):
    """The operator's output is within eight standard deviations of its roundings.

    Scores: the two planes of f32 hold an element to 2^-23 of its row's largest (uniform: 0.6 of that), so a
    product of hd of them, divided by sqrt(hd), is off by 2^-23 (Q k + q K) with Q, K the rows' largest elements and q,
    k their root mean squares; the product of two low planes, 2^-12 of their elements each, is left out
    (2^-24 q k).  The f32 sums of up to 256 products (in steps of 16) are off by 2^-24 of a partial sum each, which is
    sqrt(hd) q k at most here: 16 steps, sqrt(16) 2^-24 q k sqrt(hd) / sqrt(hd).  The f32 scale, softcap's tanh (its
    error relative to it, or 2^-22 softcap where the score is above half of softcap) and exp2: 2^-21 of the
    largest score.  16-bit rows are multiplied as they are.
    Weights of 16 bits are rounded once, by eps / 2 at most.  The f32 sums over n keys, weights and values of two
    planes: 2^-20 of the largest value.  The output is rounded once."""
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), off, softcap=softcap).cpu().double()
    f32, g = q.dtype == torch.float32, q.shape[1] // k.shape[1]
    eps = torch.finfo(q.dtype).eps / 2
    (qm, qr), (km, kr) = norms(q), norms(k)
    d = 2.0 ** -23 * (qm * kr + qr * km) + 2.0 ** -24 * qr * kr if f32 else 0.0
    x = 6 * qr * kr
    d += 4 * 2.0 ** -24 * qr * kr + 2.0 ** -21 * (min(x, softcap) if softcap else x)
    for a, b in zip(off[:-1], off[1:]):
        hidden = torch.ones(b - a, b - a, dtype=torch.bool).triu(1)
        big = v[a:b].double().abs().amax((1, 2)).cummax(0).values[:, None] if b > a else 0.0
        for h in range(q.shape[1]):
            want, by_score, by_weight = attend_bound(q[a:b, h], k[a:b, h // g], v[a:b, h // g], hidden, softcap)
            tol = 8 * (d * by_score + (0.0 if f32 else eps) * by_weight) + eps * want.abs() + 2.0 ** -20 * big
            err = (got[a:b, h] - want).abs()
            assert (err <= tol).all(), (h, float((err / tol).max()), float(err.max()))


@pytest.mark.parametrize("softcap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("lens,heads,kv,hd", [([200, 3], 4, 2, 64), ([130, 65], 2, 1, 80), ([33, 190], 8, 2, 128), ([140], 3, 1, 200),
                                              ([150, 1], 4, 2, 256)])
@pytest.mark.parametrize("name", NAMES)
def test_prompt_accuracy(gpu, name, lens, heads, kv, hd, softcap):
    dt, off = DTYPES[name], offsets(lens)
    close(rand((off[-1], heads, hd), 1, dt), rand((off[-1], kv, hd), 2, dt), rand((off[-1], kv, hd), 3, dt), off, softcap)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("name", NAMES)
def test_prompt_accuracy_sharp(gpu, name, hd):
    """Scores of some tens."""
    dt = DTYPES[name]
    close(rand((211, 4, hd), 1, dt, 3.0), rand((211, 2, hd), 2, dt, 3.0), rand((211, 2, hd), 3, dt), [0, 150, 211])


@pytest.mark.parametrize("softcap", [50.0, 4e3, 1e5, 1e6, 1e8, 1e20, 3e38])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("name", NAMES)
def test_prompt_softcap_range(gpu, name, hd, softcap):
    """A softcap far above the scores leaves them as they are."""
    dt = DTYPES[name]
    close(rand((200, 2, hd), 1, dt), rand((200, 1, hd), 2, dt), rand((200, 1, hd), 3, dt), [0, 200], softcap)


@pytest.mark.parametrize("softcap", [1e-3, 1e-20, 1e-39, 1e-45])
@pytest.mark.parametrize("name", NAMES)
def test_prompt_softcap_tiny(gpu, name, softcap):
    """One far below them leaves the weights equal (1e-3: within 2e-3 of it), zero scores included."""
    dt = DTYPES[name]
    q, k, v = rand((70, 2, 64), 1, dt), rand((70, 1, 64), 2, dt), rand((70, 1, 64), 3, dt)
    q[5], k[9] = 0.0, 0.0
    close(q, k, v, [0, 70], softcap)


def steps(n, hd, size, dt, seed):
    """q and k whose scores are c_j size^2 sqrt(hd), c_j whole numbers from -3 to 3: apart by far more than 32 bits
    round them by, or the same."""
    g = torch.Generator().manual_seed(seed)
    u = torch.randint(0, 2, (hd,), generator=g) * 2.0 - 1.0
    c = torch.randint(-3, 4, (n,), generator=g).double()
    c[:4] = torch.tensor([-3.0, -3.0, -1.0, 2.0])
    q = (size * u).expand(n, 2, hd).to(dt).contiguous()
    return q, (size * c[:, None, None] * u).to(dt).contiguous()


def largest_take_all(name, size, hd, softcap):
    """The largest scores take all the weight, in equal parts.  The weights' sum is in 32 bits, the weights of 16-bit rows
    and the output are rounded once each; those that lose are below 2^-70 (e^-50, with softcap 50)."""
    dt, n = DTYPES[name], 150
    q, k = steps(n, hd, size, dt, 5)
    v = rand((n, 1, hd), 3, dt)
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), [0, n], softcap=softcap).cpu().double()
    hidden = torch.ones(n, n, dtype=torch.bool).triu(1)
    eps = torch.finfo(dt).eps / 2
    for h in range(2):
        want = attend(q[:, h], k[:, 0], v[:, 0], hidden, softcap)
        tol = eps * want.abs() + ((0.0 if dt == torch.float32 else eps) + 2.0 ** -20) * float(v.abs().max())
        assert ((got[:, h] - want).abs() <= tol).all()


@pytest.mark.parametrize("softcap", [0.0, 50.0, 1e12])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** 7, 2.0 ** 10, 2000.0, 2.0 ** 12, 20000.0, 2.0 ** 21, 2.0 ** 40, 2.0 ** 56])
def test_prompt_large_scores_f32(gpu, size, hd, softcap):
    """Scores of any finite size."""
    largest_take_all("f32", size, hd, softcap)


@pytest.mark.parametrize("softcap", [0.0, 50.0, 1e12])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("name,size", [(t, s) for t, most in (("f16", 20000.0), ("bf16", 2.0 ** 56)) for s in
                                       (2.0 ** 7, 2.0 ** 10, 2000.0, 2.0 ** 12, 20000.0, 2.0 ** 21, 2.0 ** 40, 2.0 ** 56) if s <= most])
def test_prompt_large_scores(gpu, name, size, hd, softcap):
    """Scores of any finite size, of 16-bit rows."""
    largest_take_all(name, size, hd, softcap)


@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("name", NAMES)
def test_prompt_infinite_keys(gpu, name, hd, softcap):
    """A key with infinities that a row sees: a score of -inf takes no weight, one of +inf makes the row NaN, and softcap
    makes both finite; the key's finite elements of any size change nothing."""
    dt, n = DTYPES[name], 140
    q, k, v = rand((n, 4, hd), 1, dt), rand((n, 2, hd), 2, dt), rand((n, 2, hd), 3, dt)
    for i, at in enumerate((0, 3, 50, 99, 139)):
        k[at, 0, (7 * i) % hd] = float("-inf") if i % 2 else float("inf")
    k[50, 0, 5] = 60000.0
    k[99, 1, hd - 1] = float("nan")
    got = attn_prompt(q.cuda(), k.cuda(), v.cuda(), [0, 100, n], softcap=softcap).cpu().double()
    eps = torch.finfo(dt).eps / 2
    some = False
    for a, b in ((0, 100), (100, n)):
        hidden = torch.ones(b - a, b - a, dtype=torch.bool).triu(1)
        for h in range(4):
            kh = k[a:b, h // 2].double()
            x = q[a:b, h].double() @ torch.where(kh.isfinite(), kh, 0.0).T
            for j in (~kh.isfinite()).any(-1).nonzero()[:, 0].tolist():  # (0 times infinity nowhere: q has no zeros)
                bad = ~kh[j].isfinite()
                x[:, j] = (q[a:b, h].double()[:, bad] * kh[j, bad]).sum(-1)
            x = x / hd ** 0.5
            x = softcap * torch.tanh(x / softcap) if softcap else x
            p = torch.softmax(x.masked_fill(hidden, float("-inf")), -1)
            want = p @ v[a:b, h // 2].double()
            assert torch.equal(got[a:b, h].isnan(), want.isnan())
            fine = ~want.isnan()
            some |= bool(fine[60:].any())
            # close()'s for rows of unit variance: f32 scores off by 2^-21 (its d below 5e-7), 16-bit weights by eps,
            # eight standard deviations of each, values below 5
            tol = 8 * (2.0 ** -21 + (0.0 if dt == torch.float32 else eps)) * 5 + eps * 5
            assert ((got[a:b, h] - want).abs()[fine] <= tol).all()
    assert some


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_f32_whole_range(gpu, hd):
    """f32 rows of any normal size: queries of 1e35 against keys of 1e-35, values of 1e-36, keep their bits."""
    q, k, v = rand((150, 2, hd), 1), rand((150, 1, hd), 2), rand((150, 1, hd), 3)
    for up in (1e35, 1e-35):
        close(q * up, k / up, v, [0, 150])
    close(q, k, v * 1e-36, [0, 150])
    close(q, k, v * 1e37, [0, 150])
