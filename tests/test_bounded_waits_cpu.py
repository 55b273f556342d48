"""Bounded waits of kernels that start while the one in front still runs, read from the sources: how long a launch stays resident before
its turn, and how long its own work takes, is not its waits' affair."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashrt_b200", "csrc")
WAIT = r"tc::(?:mbar|warp)_wait\w*\("


def source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def block(text, at):
    """The braces that open behind `at`, with what is between them."""
    start = i = text.index("{", at)
    depth = 0
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            return text[start:i]


@pytest.mark.parametrize("name", ["gemm_fp8_block.cu", "sampling.cu"])
def test_every_wait_has_a_limit_of_its_own(name):
    text = source(name)
    assert "DEADLINE" not in text and "wait_until" not in text and "deadline" not in text
    waits = re.findall(WAIT, text)
    assert waits and all("_limited(" in w for w in waits)


def test_roles_of_the_block_scaled_products_wait_behind_the_kernel_in_front():
    text = source("gemm_fp8_block.cu")
    roles = 0
    for kernel in ("gemm_fp8_block_lane_kernel", "gemm_fp8_block_tile_kernel"):
        body = block(text, text.index(kernel))
        for m in re.finditer(r"if \([^{;]*warp[^{;]*\) \{|else \{", body):
            role = block(body, m.start())
            first = re.search(WAIT, role)
            if first:
                assert 0 <= role.find("pdl_wait();") < first.start(), (kernel, m.group())
                roles += 1
    assert roles == 8                                      # two kernels: producer, issuer, scales, epilogue


@pytest.mark.parametrize("kernel", ["softmax_rows_kernel", "verify_drafts_kernel"])
def test_probabilities_and_verification_wait_behind_the_kernel_in_front(kernel):
    text = source("sampling.cu")
    body = block(text, text.index(kernel + "("))
    assert 0 <= body.find("pdl_wait();") < re.search(WAIT, body).start()


def test_a_wait_that_gave_up_ends_its_warp_in_probabilities_and_verification():
    """Nothing is asked for or sent behind a wait that gave up: its warp writes the status word, stays for a bounded time, in which what is
    on its way lands before the shared memory is another's, and leaves; looked at by whole warps, since collectives follow."""
    text = source("sampling.cu")
    end = block(text, text.index("void gave_up("))
    assert re.search(r"atomicCAS\(status, 0, code\);.*until = tc::global_timer_ns\(\) \+ \d+ull;\s*while \(tc::global_timer_ns\(\) < until\) \{\}", end, re.S)
    for kernel, n in (("softmax_rows_kernel", 2), ("verify_drafts_kernel", 1)):
        body = block(text, text.index(kernel + "("))
        waits = re.findall(r"!tc::warp_wait_limited\([^;]*\)\) return gave_up\(\w+\.status, ERR_\w+\);", body)
        assert len(waits) == len(re.findall(WAIT, body)) == n
        assert not re.search(r"if \([^;]*(?:tid|lane|warp) [=<][^;]*" + WAIT, body)      # by every warp, not behind a choice of some


@pytest.mark.parametrize("name,kernel", [("gemm_fp8_block.cu", "gemm_fp8_block_lane_kernel"), ("gemm_int8.cu", "gemm_int8_lane_kernel")])
def test_tensor_memory_goes_back_before_a_cta_waits_for_its_peers(name, kernel):
    """Two CTAs an SM: a cluster whose one CTA waits for columns that another kernel's cluster holds, while its other CTA holds columns which that
    cluster's other CTA waits for, would never end, since neither the allocation nor the cluster's barrier has a limit."""
    text = source(name)
    body = block(text, text.index(kernel + "("))
    shared = block(body, body.rindex("if (S > 1) {"))
    # the warps that read it say so and arrive; the issuer arrives, waits for them, frees it, and waits for the peers only then
    order = [r"if \(warp >= \d\) asm volatile\(\"barrier\.cta\.arrive 1,", r"cluster_arrive\(\);", r"if \(warp == 1\) \{\s*asm volatile\(\"barrier\.cta\.sync 1,",
             r"if \(\*abort_flag\) let_copies_land\(\);\s*(?:tmem_give<1>|tc::tmem_dealloc)\(", r"cluster_wait\(\);", r"cluster_sync_all\(\);"]
    places = [re.search(o, shared).start() for o in order]
    assert places == sorted(places) and shared.count("cluster_sync_all();") == shared.count("cluster_wait();") == 1
    assert re.search(r"if \(S > 1\) return;.*__syncthreads\(\);.*if \(warp == 1\) (?:tmem_give<1>|tc::tmem_dealloc)\(", body, re.S)
    counts = re.findall(r'barrier\.cta\.(?:arrive|sync) 1, %0;" ::"n"\((.*?)\) : "memory"', shared)
    assert len(counts) == 2 and len(set(counts)) == 1
