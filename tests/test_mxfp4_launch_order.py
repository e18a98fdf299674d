"""What kernels that begin before the one in front of them has ended may do, and when, held to the sources: a breach shows on a GPU only
where the timing is unlucky."""

from tests.cuda_sources import kernels, source


def test_the_experts_second_half_finds_final_ids():
    """It reads the ids in front of its wait, so the first half lets it come only when the kernels before the first half have ended; and
    it reads them where every SM sees the same."""
    body = kernels("mxfp4_few.cu")["few_kernel"][1]
    assert body.index("if (KIND != SECOND) chain_wait();") < body.index("chain_next();")
    text = source("mxfp4_few.cu")
    assert "ids[" not in text and "ld.relaxed.gpu.global.s32" in text
