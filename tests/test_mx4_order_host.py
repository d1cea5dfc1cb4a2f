"""What orders the CTAs of a cluster in the 4-bit products, read in the source: no run can show an order that happens to hold.

PTX gives an mbarrier operation without a scope the scope of its own CTA.  Where the thread on the other side is in another CTA, an arrival has to
release and a wait to acquire at cluster scope, and who leaves the kernel has to know that nobody still reads or arrives at his shared memory.
"""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "mpserve_b200" / "csrc"
TENSOR, LINEAR = ((CSRC / name).read_text() for name in ("mx4_tensor.cuh", "mx4_linear.cu"))


def _kernel(name):
    return LINEAR.split(f"\n{name}(", 1)[1].split("\n}\n", 1)[0]


def test_arrivals_in_another_cta_release_at_cluster_scope():
    arrivals = re.findall(r"mbarrier\.arrive\S*", TENSOR)
    remote = [a for a in arrivals if "multicast" not in a and "shared::cluster" in a and "::one" not in a]
    assert remote and all(".release.cluster." in a for a in remote)


def test_waits_for_another_cta_acquire_at_cluster_scope():
    assert re.search(r"mbarrier\.try_wait\.parity\.acquire\.cluster\.shared::cta\.b64", TENSOR)
    assert "warp_wait<true>(received" in _kernel("mx4_stream_kernel")
    wide = _kernel("mx4_wide_kernel")
    # the first CTA's waits for the second one's arrivals, and both CTAs' for what the first one's multiplications arrive at
    waits = re.findall(r"(?:bar|warp)_wait(<true>)?\((\w+)", wide)
    assert {bar for _, bar in waits} == {"empty", "full", "acc_empty", "acc_full", "drained"}
    assert all(scope for scope, bar in waits if bar in ("empty", "acc_empty", "acc_full"))
    assert "warp_wait<true>(full(s)" in wide
    # bounded waits begin when what they wait for is under way: the end of all multiplications is waited for by who issued them, and told to nobody else
    assert "tensor_commit_pair<1>(lead, drained);" in wide
    assert wide.index("if (rank == 0) {\n            const uint32_t lead") < wide.index("drained, 0, &failed")


def test_copies_of_a_pair_count_at_the_barrier_that_is_waited_at():
    """An untiled copy counts at its own CTA's barriers; nothing may stand between a copy and the thread that multiplies what it brings."""
    wide = _kernel("mx4_wide_kernel")
    assert "bulk_g2s(" not in wide and "tiled_g2s_pair(" in wide
    assert re.search(r"bar = peer_address\(full\(s\), 0\)", wide)


def test_nobody_leaves_behind_an_arrival_that_orders_nothing():
    assert re.search(r"cluster_sync\(\);[^\n]*until both are done", _kernel("mx4_wide_kernel"))
    assert re.search(r"cluster_sync\(\);[^\n]*nobody leaves while his part is read", _kernel("mx4_stream_kernel"))
    body = TENSOR.split("void cluster_sync()", 1)[1].split("\n}\n", 1)[0]
    assert "barrier.cluster.arrive.release" in body and "barrier.cluster.wait.acquire" in body
