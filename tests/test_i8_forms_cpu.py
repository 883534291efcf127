"""The table of what every form of the 8-bit integer products takes, and the figures in the source that choose among them: made for each other."""
import re

import numpy as np

from perf import inner_i8_forms as forms


def test_the_table_has_the_forms_of_the_source():
    with open(forms.TABLE) as f:
        headings = dict(line.rstrip("\n").split(": ", 1) for line in f if re.match(r"products.*: 1 rows<", line))
    assert list(headings) == [name for name, _, _ in forms.SECTIONS]
    for name, by_experts, _ in forms.SECTIONS:
        listed = forms.forms(by_experts)
        assert headings[name] == ", ".join("%d %s" % (i + 1, f.name) for i, f in enumerate(listed))
    for at, shape, rule, times in forms.read():
        listed = forms.forms(forms.SECTIONS[at][1])
        assert len(times) == len(listed) and rule is not None and times[forms.chosen(listed, shape)[0]] is not None, shape


def test_the_figures_choose_as_the_comment_beside_them_says():
    for at, (name, by_experts, fitted) in enumerate(forms.SECTIONS):
        shapes, us = forms.timed_shapes(at)
        listed = forms.forms(by_experts)
        longer = np.array([us[i, forms.chosen(listed, s)[0]] for i, s in enumerate(shapes)]) / us.min(1) - 1
        inside = "outside" not in name
        assert longer.mean() < (0.02 if inside else 0.08) and longer.max() < (0.30 if inside else 0.80), name
