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


def test_results_of_the_kernel_in_front_are_not_read_through_the_read_only_path():
    """A `const __restrict__` pointer lets the compiler read early and through the read-only path, whatever stands between. The quantiser
    and its way back begin when everything in front of them has ended."""
    for name in ("mxfp4_few.cu", "mxfp4_route.cu", "mxfp4_tc.cu"):
        assert "__restrict__" not in source(name) and "__ldg" not in source(name) and "pair_weight" not in source(name)
        for kernel, (parameters, body) in kernels(name).items():
            assert "chain_wait();" in body, kernel
    for kernel, (parameters, body) in kernels("mxfp4.cu").items():
        assert "chain" not in body
    assert "launch_behind" not in source("mxfp4.cu") and "cudaLaunchKernelEx" not in source("mxfp4.cu")


def test_the_next_kernel_comes_when_this_one_has_its_tensor_memory():
    """A kernel that begins early may take tensor memory before it waits for this one's end. What it took a CTA here would wait for, for good."""
    found = 0
    for kernel, (parameters, body) in kernels("mxfp4_tc.cu").items():
        assert body.count("chain_next();") == 1
        taken = body.index("__syncthreads();", body.index("tcgen05.alloc"))
        assert taken < body.index("chain_next();"), kernel
        found += 1
    assert found == 2


def test_a_layer_of_experts_begins_when_everything_in_front_of_it_has_ended():
    """With all launches chained, the products behind the plan would else take tensor memory while a kernel in front of the plan, that has yet
    to take its own, waits."""
    body = kernels("mxfp4_route.cu")["plan_kernel"][1]
    assert body.index("chain_wait();") < body.index("chain_next();")
