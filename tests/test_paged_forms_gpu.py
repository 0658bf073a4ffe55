"""Every launch that paged_attention can make (paged_forms.FORMS; test_paged_plan_cpu.py holds these shapes to it), over pages
of 16 and of 64 rows, without and with bias, also where keys are hidden, against float64.  Tolerances as in test_paged_gpu."""
import math

import pytest

from paged_forms import FORMS
from paged_util import slots_of
from tests.test_paged_gpu import _attention, _normal_bias

pytestmark = pytest.mark.gpu
forms = pytest.mark.parametrize("form", FORMS, ids=[f.name for f in FORMS])
pages = pytest.mark.parametrize("page", [16, 64])


@forms
@pages
@pytest.mark.parametrize("bias", [False, True])
def test_form(form, page, bias):
    _attention(form.new, form.used, form.H, form.Hkv, page, bias=_normal_bias if bias else None, seed=page)


@forms
@pages
@pytest.mark.parametrize("bias", [False, True])
def test_form_with_hidden_keys(form, page, bias):
    """Entries of no page in every fifth sequence; with bias, keys hidden from all heads by -inf whose rows are no numbers in
    the next."""
    dead = [(b, j) for b, u in enumerate(form.used) if b % 5 == (1 if len(form.used) > 1 else 0) for j in range(0, u, 37)]

    def hide(g, B, H, n):
        x = _normal_bias(g, B, H, n)
        for b in sorted({b for b, _ in dead}):
            x[b, :, [j for s, j in dead if s == b]] = -math.inf
        return x

    def prepare(cache, table, b):
        if b is not None:
            at = slots_of(table, page, dead).long()
            cache.k[at // page, :, at % page] = math.nan
            cache.v[at // page, :, at % page] = math.inf
        for s in range(0, len(form.used), 5):
            n = (form.used[s] + page - 1) // page
            table[s, n // 2] = -1
            table[s, n // 3:n // 3 + n // 8] = cache.n_pages

    _attention(form.new, form.used, form.H, form.Hkv, page, bias=hide if bias else None, seed=page + 1, prepare=prepare)


@forms
@pages
@pytest.mark.parametrize("bias", [False, True])
def test_form_with_large_values(form, page, bias):
    """Values near the largest float, of one sign in a KV head so that their sums grow with the keys: outputs are averages of
    them, and finite."""
    def prepare(cache, table, _):
        cache.v.copy_((cache.v.abs() * 1.5e38).clamp(max=3.3e38))
        cache.v[:, 1::2].neg_()
    _attention(form.new, form.used, form.H, form.Hkv, page, bias=_normal_bias if bias else None, seed=page + 2, prepare=prepare)
