"""Kernels whose blocks wait for each other in a cluster while they hold tensor memory: two such blocks on one processor must never wait for each other's
columns, or both clusters wait for ever.  Read from the sources (such a wait is not tried out on a GPU)."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xinfer_b200", "csrc")
PROCESSOR, BLOCK = 228 * 1024, 1024          # shared memory of a processor, and what a block takes of it beside its own
COLUMNS = 512


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def constants(text):
    values = {}
    for group in re.findall(r"constexpr int ([^;{}()]*);", text):
        for name, value in re.findall(r"(\w+) = ([\w *+]+)", group):
            if re.fullmatch(r"[\w *+]+", value):
                try:
                    values[name] = eval(value, {}, values)
                except NameError:
                    pass
    return values


def smallest_skinny_block(tokens):
    """Shared memory of a block of gemm_skinny_tc.cu with others in its cluster: two stages, or its sums."""
    c = constants(source("gemm_skinny_tc.cu"))
    stage = (c["TILE_N"] + tokens) * c["TILE_K"] * 2
    return max(2 * stage, tokens * c["TILE_N"] * 4) + 1024


def test_which_kernels_have_both():
    both = [os.path.basename(f) for f in sorted(glob.glob(os.path.join(CSRC, "*.cu")))
            if re.search(r"tcgen05\.alloc|\btmem_alloc\s*\(", source(os.path.basename(f))) and "cudaLaunchAttributeClusterDimension" in source(os.path.basename(f))]
    assert both == ["gemm_skinny_tc.cu", "linear4_tc.cu"]          # (another one has to be looked at here)


def test_blocks_of_few_columns_always_find_theirs():
    # gemm_skinny_tc.cu: columns for the shared memory that its blocks take, whatever their mixture on a processor
    for tokens in (16, 32, 64, 128, 256):
        assert max(32, tokens) / (smallest_skinny_block(tokens) + BLOCK) < COLUMNS / PROCESSOR


def test_a_block_that_takes_all_columns_is_alone():
    text = source("linear4_tc.cu")
    c = constants(text)
    assert re.search(r"smem = splits > 1 && holds < SMEM_CLUSTERED \? SMEM_CLUSTERED : holds;", text) and re.search(r"dynamicSmemBytes = smem;", text)
    left = PROCESSOR - BLOCK - c["SMEM_CLUSTERED"]
    smallest_own = 4 * 2 * 32 * 128            # (four stages of 32 tokens, of blocks that are in no cluster)
    assert left < min(smallest_skinny_block(16), smallest_own) + BLOCK
    assert c["SMEM_CLUSTERED"] <= c["SMEM_MOST"] <= 227 * 1024 - 1024
