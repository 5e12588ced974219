"""The sampler's CTAs write into one another's shared memory.  That is allowed once every CTA of the cluster has started,
so a barrier of the cluster has to lie before the first such access.  Nothing on the GPU shows its absence (the CTAs of a
cluster nearly always start together), so the order is read from the kernel's source.
"""

from __future__ import annotations

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kappa_b200", "csrc")

# What reaches into another CTA: the accesses themselves, and the members of Row that make them.
REMOTE = r"\b(?:R\.(?:publish|reduce|reduce_all|prefix|sum|sync)|mapa_shared|st_cluster_u\d+|ld_cluster_u\d+)\s*\("


def _kernel(name: str, file: str) -> str:
    src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, file)).read())
    at = re.search(rf"__global__[^;{{]*\b{name}\s*\(", src)
    assert at, f"{name} is not in {file}"
    i = src.index("{", at.end())
    depth, j = 1, i + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(src[j], 0)
        j += 1
    return src[i:j]


def test_the_sampler_waits_for_its_cluster_before_the_first_remote_access():
    body = _kernel("sample_kernel", "sample.cu")
    first = re.search(REMOTE, body)
    assert first, "the kernel makes no remote access"
    arrive = re.search(r"if \(ranks > 1\) cluster_arrive_relaxed\(\);", body)
    wait = re.search(r"if \(ranks > 1\) \{\s*__syncwarp\(\);\s*cluster_wait\(\);\s*\}", body)
    assert arrive and wait, "no barrier of the cluster's start"
    assert arrive.start() < wait.start() < first.start()


def test_the_pair_kernels_start_with_a_barrier_of_the_pair():
    for name, file in (("linear_q8_pair_kernel", "gemm_q8.cu"), ("w8_gemm_tc2_kernel", "gemm_tc2.cu")):
        body = _kernel(name, file)
        first = re.search(r"\b(?:mapa_shared|mbar_arrive_cluster|tma_load_\dd_pair|mma_commit_pair)\s*\(", body)
        barrier = re.search(r"\bcluster_sync_all\(\);", body)
        assert first and barrier and barrier.start() < first.start()


def test_the_split_linear_reads_other_ctas_behind_a_barrier():
    body = _kernel("linear_q8_kernel", "gemm_q8.cu")
    first = re.search(r"\bmapa_shared\s*\(", body)
    barrier = re.search(r"\bcluster_sync_all\(\);", body)
    assert first and barrier and barrier.start() < first.start()
