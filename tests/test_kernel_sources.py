"""Rules that the kernel sources have to keep and that no run shows reliably (CPU only)."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "expertscattergather_b200", "csrc")


def _kernels():
    """(file, name, parameters, body) of every kernel."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__\s+void\s", text):
            k = re.compile(r"(\w+_kernel\w*)\s*\(").search(text, m.end())
            i = k.end()
            j = text.index("{", i)
            depth, end = 1, j + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            yield os.path.basename(path), k.group(1), text[i:j], text[j:end]


KERNELS = list(_kernels())


def test_kernels_are_found():
    names = {k[1] for k in KERNELS}
    assert {"strict_kernel", "dense16_kernel", "generic_rowgemm_kernel", "scatter_prepare_kernel", "csr_batch_place_kernel"} <= names


DEPENDENTS = [k for k in KERNELS if "pdl_wait" in k[3]]


@pytest.mark.parametrize("kernel", DEPENDENTS, ids=[k[1] for k in DEPENDENTS])
def test_dependent_kernels_promise_nothing_about_aliases(kernel):
    """A kernel that may start under the one before it must not tell the compiler that nobody writes its inputs meanwhile: loads
    through `__restrict__` pointers are not bound by the wait."""
    file, name, params, body = kernel
    assert "__restrict__" not in params + body, f"{file}: {name}"


def test_ctas_that_count_for_themselves_are_resident_together():
    """The grid of the kernel that counts ids and fills has four CTAs for an SM; one that has to wait for the others counts and fills after them."""
    text = open(os.path.join(CSRC, "egs_generic.cu")).read()
    assert re.search(r"__launch_bounds__\(kPrepThreads, 4\)\s+scatter_prepare_kernel", text)
    assert "size_t grid = 4 * 148;" in text


def test_arrivals_at_another_ctas_barrier_name_their_scope():
    """An arrival without one orders memory for its own CTA alone; what it announces to another CTA may not be there yet."""
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        for at in re.findall(r"mbarrier\.arrive[\w.:]*", re.sub(r"//[^\n]*", "", open(path).read())):
            if "shared::cluster" in at:
                found += 1
                assert ".release.cluster." in at or ".relaxed.cluster." in at, f"{os.path.basename(path)}: {at}"
    assert found >= 2


def test_scales_of_a_pair_are_waited_for_at_the_scope_they_are_released_at():
    """The leader's tensor core reads both CTAs' scales and tiles: its waits for them acquire what the other CTA has released."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "egs_fp4_tensor.cu")).read())
    issuer = text[text.index("warp == kIssueWarp", text.index("warp == kBoxWarp")):text.index("warp < kReadWarp0")]
    for barrier in ("scale_full", "full", "smem_u32(&hdr->acc_empty[buf])"):
        assert f"mbar_wait_all<PAIR>({barrier}," in issuer
    assert re.search(r"mbar_wait_all\(smem_u32\(&hdr->scale_stored\[.*\n.*mbar_arrive_cluster\(map_to_cta\(smem_u32\(&hdr->scale_full", issuer)
