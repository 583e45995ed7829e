"""wzy_sample (include/wzy_paged.h): top-k between the groups' and the row's forms, and flat rows, against 64 bits."""
import numpy as np
import pytest

from mx_ref import BF16, F16, F32
from test_gpu_paged import check_sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("vocab,gap", [(2049, 0), (8193, 3), (33333, 7), (151936, 0)])
@pytest.mark.parametrize("filters", ["k", "kp", "km", "kpm"])
def test_sample_middle_top_k(wz, gpu, t, vocab, gap, filters):
    rng = np.random.default_rng(vocab + len(filters))
    k = np.array([127, 128, 129, 500, 2047, 2048, 2049, 2048])
    x = rng.standard_normal((8, vocab)) * np.array([[3.0], [1.0], [3.0], [1.0], [2.0], [3.0], [1.0], [0.05]])
    p = dict(temp=rng.uniform(0.3, 1.5, 8), top_k=k, u=rng.random(8).astype(np.float32))
    if "p" in filters:
        p["top_p"] = rng.choice([0.3, 0.9, 0.999], 8)
    if "m" in filters:
        p["min_p"] = rng.choice([1e-4, 0.05, 0.3], 8)
    check_sample(wz, x, t, gap, **p)


@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_sample_ties_at_the_last_of_top_k(wz, gpu, t):
    # a few large logits, then hundreds or thousands of equal ones around the k-th place: the lower ids remain
    rng = np.random.default_rng(5)
    n, k = 40000, np.array([129, 300, 1000, 2048, 2048, 700])
    x = rng.standard_normal((6, n)) - 6.0
    for r, (large, equal) in enumerate([(100, 50), (100, 4000), (990, 300), (2000, 3000), (1, 9000), (699, 2)]):
        at = rng.choice(n, large + equal, replace=False)
        x[r, at[:large]] = 4.0 + np.round(rng.standard_normal(large), 2)
        x[r, at[large:]] = 0.5
    for u in (0.0, 0.5, 0.97, 1.0):
        check_sample(wz, x, t, temp=np.full(6, 0.9), top_k=k, u=np.full(6, u, np.float32))
        check_sample(wz, x, t, temp=np.full(6, 3.0), top_k=k, top_p=np.full(6, 0.9), min_p=np.full(6, 0.01), u=np.full(6, u, np.float32))


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("sd,temp", [(1.5, 1.5), (2.5, 2.0), (0.2, 1.0), (0.01, 5.0)])
def test_sample_flat_rows(wz, gpu, t, sd, temp):
    # bins of thousands of different logits: more than are gathered
    rng = np.random.default_rng(int(100 * sd))
    x = rng.standard_normal((6, 151936)) * sd
    u = rng.random(6).astype(np.float32)
    check_sample(wz, x, t, temp=np.full(6, temp), top_p=np.full(6, 0.95), u=u)
    check_sample(wz, x, t, temp=np.full(6, temp), top_k=np.full(6, 5000), min_p=np.full(6, 0.01), u=u)
