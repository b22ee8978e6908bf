"""Rules of the cluster kernel of the gated linear recurrence that a GPU run cannot show to be broken, checked in its source."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "t2fw_b200", "csrc")


def _kernel():
    with open(os.path.join(CSRC, "glr_scan.cuh")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    start = text.index("glr_scan_kernel(const ScanArgs<T> p) {")
    depth, i = 0, text.index("{", start)
    for j in range(i, len(text)):
        depth += {"{": 1, "}": -1}.get(text[j], 0)
        if depth == 0:
            return text[i:j + 1]
    raise AssertionError("unbalanced braces")


def test_waits_for_the_kernel_before_it_first():
    """It is launched to start before that one has ended: one unconditional wait, before anything is read."""
    body = _kernel()
    assert body.count("dependency_wait()") == 1
    before = body[:body.index("dependency_wait()")]
    assert before.count("{") - before.count("}") == 1 and "[" not in re.sub(r"\b\w+(\[[^\]]*\])+;", "", before)


def test_every_thread_reaches_the_cluster_barriers():
    """Blocks meet once before they send (all threads) and once before they leave: the last warp on its own way out, the others
    on theirs; nothing else returns."""
    body = _kernel()
    assert body.count("if (C > 1) cluster_sync();") == 2 and body.count("cluster_sync()") == 3
    first = body.index("cluster_sync()")
    assert first < body.index("if (warp == kWarps)")
    assert len(re.findall(r"\breturn;", body)) == 1
    assert re.search(r"if \(C > 1\) cluster_sync\(\);\s*return;\s*\}", body)


def test_named_barriers_count_the_same_threads():
    """The warps report where the last one meets and the other way round, with the same count; no block barrier is left that
    one side would miss."""
    body = _kernel()
    calls = re.findall(r"\b(report|meet)<([^>]*)>\((kMaps|kIns)", body)
    assert sorted((c[0], c[2]) for c in calls) == [("meet", "kIns"), ("meet", "kMaps"), ("report", "kIns"), ("report", "kMaps")]
    assert {c[1] for c in calls} == {"kThreads + 32"}
    assert "__syncthreads" not in body
