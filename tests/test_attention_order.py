"""CPU: orderings that the attention kernels' correctness rests on and that no run on a GPU can show to be missing, checked in
their source."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "fastkernels_b200" / "csrc"


def code(name):
    """A kernel file without its comments."""
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", ["attention_few.cu", "attention_tile.cu"])
def test_the_plan_is_fenced_from_the_copies_that_take_its_memory(name):
    """The plan is written and read in the ring's memory by ordinary accesses; tensor copies, which belong to the async proxy, write there
    next.  A barrier alone does not order the two proxies: every thread has to fence before it."""
    after = code(name).split("locate(p, run0, upto, room", 1)[1]
    assert "fence_async_proxy();" in after.split("__syncthreads();", 1)[0]


@pytest.mark.parametrize("name", ["attention_few.cu", "attention_tile.cu"])
def test_a_warp_decides_together_whether_a_barrier_has_passed(name):
    """A barrier's phase may change between the looks of two lanes.  What depends on a look and is done by the whole warp (announcing the
    loads of all lanes) needs one answer for all of them."""
    looks = [m.start() for m in re.finditer(r"mbar_(?:try|test)_wait\(", code(name))]
    assert all(code(name)[:at].rstrip().endswith("__all_sync(kFull,") for at in looks)


def test_every_wait_of_a_pair_reaches_both_blocks_and_stops_what_follows():
    """Blocks of a pair depend on each other: when a wait of one gives up, the other must learn of it, nothing more may be issued or announced,
    and neither block may leave while something is on its way to it."""
    text = code("attention_tile.cu")
    assert text.count("warp_wait(") == 2 and "mbar_wait" not in text                          # the place that tells the other block, and one that ends there
    given_up = text.split("warp_wait(", 1)[1].split("return false;", 1)[0]
    assert "bar.abort_flag = 1;" in given_up and "tell_other_block(&bar.abort_flag);" in given_up
    assert "return wait(b, parity);" in text.split("warp_wait(", 2)[2].split("};", 1)[0]
    assert "%%cluster_ctarank" in text and "st.shared::cluster" in text.split("void tell_other_block", 1)[1].split("}\n", 1)[0]
    waits = re.findall(r"([^\n;{}]*)\bwait(?:_long)?\(&?b", text)
    assert waits and all(re.search(r"(=|!|&&|return) *\(?$", w) for w in waits)               # no answer is thrown away
    assert all("!dead()" in line for line in re.findall(r"[^\n]*arrive_first\(&bar[^\n]*", text))
    assert text.rindex("linger();") < text.rindex("cluster_sync();") < text.rindex("pair_tmem_dealloc(tmem)")
