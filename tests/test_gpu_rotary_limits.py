"""Rotation at the ends of its ranges: elements and pairs that stay as they are, positions up to 2^32,
heads whose squares leave FP32."""
from decimal import Decimal, getcontext

import numpy as np
import pytest

import layer_util as L
import turbo_decode_tail as T
from test_gpu_layer_cache import code, ids, tensor

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def turned(r, x, pos, dtype="f32"):
    xt = tensor(x, dtype)
    out = torch.empty_like(xt)
    r.apply(r.make_inputs(x.shape[0], dtype=code(dtype), q=xt, q_heads=x.shape[1], positions=ids(pos), q_out=out))
    return out.float().cpu().numpy()


@pytest.mark.parametrize("dim,rotary", [(64, 32), (128, 16), (256, 128), (512, 64)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_elements_past_the_rotation_pass_as_they_are(dtype, pairs, dim, rotary):
    """Infinities and NaN among them too, and their neighbours."""
    rng = np.random.default_rng(1)
    x = L.bf16(rng.standard_normal((5, 3, dim)).astype(np.float32))
    x[0, 0, rotary], x[1, 1, dim - 1], x[2, 2, rotary + 9], x[3, 0, rotary + 4] = np.inf, -np.inf, np.nan, -0.0
    r = T.Rotary(dim, rotary_dim=rotary, layout=int(pairs), norms=0)
    got = turned(r, x, np.arange(5) * 1000 + 7, dtype)
    assert np.array_equal(got[..., rotary:].view(np.uint32) << 1 >> 23, x[..., rotary:].view(np.uint32) << 1 >> 23)  # NaN too
    same = ~np.isnan(x[..., rotary:])
    assert np.array_equal(got[..., rotary:][same].view(np.uint32), x[..., rotary:][same].view(np.uint32))
    assert np.isfinite(got[..., :rotary]).all()


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pairs_of_frequency_zero_stay_as_they_are(dtype, pairs):
    rng = np.random.default_rng(2)
    dim = 128
    f = rng.uniform(0.1, 2, dim // 2)
    f[::5] = 0.0
    x = L.bf16(rng.standard_normal((4, 2, dim)).astype(np.float32))
    first = (np.arange(0, 64, 5) * 2) if pairs else np.arange(0, 64, 5)
    second = first + 1 if pairs else first + 64
    x[1, 0, first], x[2, 1, second] = np.inf, -np.inf
    r = T.Rotary(dim, inv_freq=f, layout=int(pairs), norms=0)
    got = turned(r, x, np.array([0, 5, 10**9, 2**32 - 1], np.uint32), dtype)
    still = np.concatenate([first, second])
    assert np.array_equal(got[..., still].view(np.uint32), x[..., still].view(np.uint32))
    assert np.isfinite(np.delete(got, still, axis=2)).all()


@pytest.mark.parametrize("theta", [1e4, 5e5, 1e6])
def test_angles_of_far_positions(theta):
    """(1, 0) turned is (cos, sin). The angle is within 2^-31 turns of position * theta^(-2 i / R), in
    decimal arithmetic of 60 digits; sine and cosine add 4 roundings of themselves."""
    getcontext().prec = 60
    two_pi = Decimal("6.28318530717958647692528676655900576839433879875021164194988918")
    rng = np.random.default_rng(3)
    dim, n = 64, 400
    pos = rng.integers(2**32 - 2**30, 2**32, n, dtype=np.uint64).astype(np.uint32)
    pos[0] = 2**32 - 1
    x = np.zeros((n, 1, dim), np.float32)
    x[..., :dim // 2] = 1.0
    got = turned(T.Rotary(dim, theta=theta, norms=0), x, pos)[:, 0].astype(np.float64)
    turn = np.empty((n, dim // 2))
    for i in range(dim // 2):
        per = Decimal(theta) ** (Decimal(-2 * i) / Decimal(dim)) / two_pi
        turn[:, i] = [float((int(p) * per) % 1) for p in pos]
    angle = 2 * np.pi * turn
    want = np.concatenate([np.cos(angle), np.sin(angle)], axis=1)
    bound = 2 * np.pi * 2.0**-31 + 4 * 2.0**-24 * np.abs(want)
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norms_of_heads_whose_squares_leave_the_type(dtype, dim):
    """Heads of 1e-30 to 1e38 with eps 0, tokens of all sizes in one call: 14 roundings of the mean's terms and
    sum, halved by the root, and 7 of root, division, powers of two and products."""
    rng = np.random.default_rng(4)
    size = np.array([1e-30, 1e-22, 1e-10, 1.0, 1e10, 1e19, 1e25, 1e37], np.float32)
    x = (rng.uniform(0.1, 1, (8, 3, dim)) * rng.choice([-1, 1], (8, 3, dim)) * size[:, None, None]).astype(np.float32)
    x[4, 1] *= np.float32(1e15)  # and of one call's heads
    x = L.bf16(x) if dtype == "bf16" else x
    r = T.Rotary(dim, rotary_dim=0, eps=0.0)
    got = turned(r, x, np.zeros(8, np.uint32), dtype)
    want = L.norm(x, 0.0)
    bound = 14 * 2.0**-24 * np.abs(want)
    bound += 2.0**-8 * (np.abs(want) + bound) if dtype == "bf16" else 0.0
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())
    plain = np.array(x)
    plain[[0, 1, 5, 6, 7]], plain[4, 1] = 1.0, 1.0
    pos = np.arange(5, 13)
    for r in (r, T.Rotary(dim, eps=0.0), T.Rotary(dim, eps=0.0, rotary_dim=32, layout=T.TURBO_ROPE_PAIRS)):
        got, again = turned(r, x, pos, dtype), turned(r, plain, pos, dtype)  # the same bits whatever stands beside them
        assert np.array_equal(again[[2, 3]], got[[2, 3]]) and np.array_equal(again[4, [0, 2]], got[4, [0, 2]])


@pytest.mark.parametrize("bits", [4, 8])
def test_normed_values_whose_squares_leave_the_type(bits):
    rng = np.random.default_rng(5)
    n, dim = 40, 128
    size = (10.0 ** rng.uniform(-35, 37, (n, 1, 1))).astype(np.float32)
    v = (rng.uniform(0.1, 1, (n, 2, dim)) * size).astype(np.float32)
    vt, pt = tensor(v, "f32"), ids(np.arange(n))
    cache = T.KvCache(2, 32, 2, dim, bits=bits)
    r = T.Rotary(dim, rotary_dim=0, norms=T.TURBO_NORM_V, eps=0.0)
    r.apply(r.make_inputs(n, k=torch.zeros_like(vt), v=vt, kv_heads=2, cache=cache, slots=pt))
    back = torch.empty_like(vt)
    cache.read(pt, n, None, back)
    want = L.norm(v, 0.0)
    # half a step of a range below 2 with its two roundings up, and the norm's 14 roundings
    g = want.reshape(n, 2, -1, 64)
    step = (g.max(-1) - g.min(-1) * (1 - 2.0**-7)) * (1 + 2.0**-7) / (2**bits - 1)
    bound = 0.5 * np.repeat(step, 64, axis=-1).reshape(want.shape) * (1 + 2.0**-12) + 14 * 2.0**-24 * np.abs(want).max(-1, keepdims=True)
    assert np.all(np.abs(back.cpu().numpy() - want) <= bound)
