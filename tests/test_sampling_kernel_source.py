"""CPU checks of the sampling kernel's source where a mistake could only show as a race on the GPU."""
import os
import re

import pytest

from conftest import ROOT


def body(name):
    """The text of a function's definition in sample.cu, by its braces."""
    text = open(os.path.join(ROOT, "swvr_b200", "csrc", "sample.cu")).read()
    text = re.sub(r"//[^\n]*", "", text)
    at = re.search(r"\b%s\([^;{]*\{" % name, text)
    i, depth = at.end(), 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
    return text[at.end():i]


def read_by_peers(text):
    return set(re.findall(r"map_shared_rank\(&s\.(\w+)", text))


def written(text):
    return set(re.findall(r"\bs\.(\w+)(?:\[[^]]*\])?\s*(?:=(?!=)|\+=)", text)) | set(re.findall(r"atomicAdd\(&s\.(\w+)", text))


def test_the_scan_finds_what_gather_does():
    assert "n_list" in read_by_peers(body("gather")) and {"n_list", "list"} <= written(body("gather"))


@pytest.mark.parametrize("after", ["choose_from_list", "sort_list", "exact_total"])
def test_nothing_that_peers_may_still_read_is_written_after_gather(after):
    """gather ends with every CTA of the cluster reading every CTA's count, and no cluster barrier follows in the CTA that
    chooses from the list: what runs there before the next barrier leaves those words alone."""
    assert not read_by_peers(body("gather")) & written(body(after))
