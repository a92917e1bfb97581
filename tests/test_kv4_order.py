"""What the kernels of the 4-bit cache may not read before, or how, since kernels in front of them may still run when they start; read off the CUDA sources."""
import os
import re

from test_kernel_order import CSRC, kernels


def test_an_ordinary_launch_stands_between_the_allocator_and_who_reads_its_row_maps_without_waiting():
    """rope_rows_kernel reads positions before it waits.  In a 4-bit batch the page allocator, a kernel of the same pass, writes them: an ordinary launch between the two
    (which begins when everything before it is complete, and behind which nothing begins sooner) is what makes that right."""
    body = kernels()["rope_rows_kernel"]
    assert body.index("p.row_pos[m]") < body.index("kernel_wait()")
    embed = re.search(r"int embed_rows_launch\(.*?\n\}", open(os.path.join(CSRC, "prefill.cu")).read(), re.S).group(0)
    assert "embed_rows_kernel<<<" in embed and "launch_after(" not in embed
    rows = re.search(r"static int batch_rows\(.*?\n\}", open(os.path.join(CSRC, "engine.cu")).read(), re.S).group(0)
    assert rows.index("batch_step4(") < rows.index("embed_rows_launch(") < rows.index("rope_kv_paged_launch(")
    assert rows.count("batch_step4(") == rows.count("embed_rows_launch(") == 1


def test_the_cache_is_not_read_as_constant_data():
    """The writer, or the kernel that makes q, may run when the attention starts: loads for data that nobody writes meanwhile are not for those."""
    for name in sorted(os.listdir(CSRC)):
        if name.startswith("kv4") or name == "page_step.cu":
            text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
            assert not re.search(r"__ldg\b|ld\.global\.nc|__restrict__", text), name
