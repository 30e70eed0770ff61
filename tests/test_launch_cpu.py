"""How the kernels' launches are written, from the source files alone.  No GPU is touched."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "okc_muse_kernels_b200", "csrc")


def test_shared_memory_limits_are_constants_of_the_kernels():
    """The limit belongs to a kernel on its device: set to a call's own size, it can be lowered by a call of another thread
    before this call's launch."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            for limit in re.findall(r"cudaFuncAttributeMaxDynamicSharedMemorySize,\s*(.+?)\);", f.read()):
                assert re.fullmatch(r"k[A-Z]\w*", limit), f"{name}: {limit}"
                found += 1
    assert found >= 10


def test_the_split_product_drains_its_copies_whichever_wait_ran_out():
    """A wait that runs out leaves copies on their way into shared memory.  In okc_int8_mid it may be the issuer's, when both
    producers have started everything and left their loops: the drain stands behind all of them, in front of the last barrier,
    and asks for the flag that every wait sets."""
    with open(os.path.join(CSRC, "int8.cu")) as f:
        body = f.read().split("okc_int8_mid(const")[1].split("static int tmem_cols_for")[0]
    tail = body[body.rindex("finish(std::integral_constant<int, 1>"):body.rindex("cluster.sync()")]
    assert re.search(r"if \(gave_up != 0\) \{[^}]*mbar_try\(full0[^}]*kWaitLimitCycles", tail)
    read = body.index("const int gave_up = abort_code;")        # behind every wait and the barrier after them
    assert body.rindex("mbar_wait") < body.index("cluster.sync()") < read < body.index("auto finish")


def test_the_streamed_norms_start_no_copy_behind_one_that_is_late():
    """Their threads stay in the loop over the rows when a wait has run out.  A slot's barrier then still counts the copy that is
    late, and another arrival on it is one too many: no further row may be fetched."""
    with open(os.path.join(CSRC, "norm.cu")) as f:
        kernels = f.read().split("__global__")
    streamed = [k for k in kernels if " okc_block_norm_stream" in k.split("{")[0]]
    assert len(streamed) == 2
    for body in streamed:
        wait = body.index("mbar_wait(")
        again = [line for line in body[wait:].splitlines() if "fetch(" in line]
        assert len(again) == 1
        own = re.search(r"const bool (\w+) = mbar_wait\(", body)          # whether this thread's wait saw the copy land
        assert "&& abort_code == 0) fetch(" in again[0] or own and f"&& {own[1]}) fetch(" in again[0]
