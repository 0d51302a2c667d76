"""What the launchers of layer normalisation, the embedding and the gradient norm refuse. A refusal
prints and exits before anything is enqueued, so it needs no GPU; each runs in a process of its own."""
import subprocess
import sys
import textwrap

import pytest

from metaphor_amd import ffi

FAKE = 0x100000000000  # an address nothing dereferences: the call ends before a launch

CASES = [
    ("layernorm_ij_j", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, 1e-5, 4, (1 << 30) + 1", "row length must not exceed"),
    ("layernorm_ij_j_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE + 512}, None, 1e-5, 0.0, 4, 64", "mpLayernormReverseScratchBytes"),
    ("layernorm_ij_j_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, 1e-5, 0.0, 4, (1 << 30) + 1", "row length must not exceed"),
    ("layernorm_ij_j_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE + 64}, 1e-5, 0.0, 4, 64", "must be different vectors"),
    ("layernorm_ij_j_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE + 512}, {FAKE + 2}, 1e-5, 0.0, 4, 64", "aligned to its sums"),
    ("layernorm_ij_j_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE}, {FAKE + 512}, {FAKE + 8}, 1e-5, 0.0, 4, 64", "16-byte aligned"),
    ("embedding_i_ij", f"{FAKE}, {FAKE}, {FAKE}, 1.0, 2, 10, 4, 64", "4 or 8 bytes wide"),
    ("embedding_i_ij", f"{FAKE}, {FAKE + 4}, {FAKE}, 1.0, 8, 10, 4, 64", "aligned to their width"),
    ("embedding_i_ij", f"{FAKE}, {FAKE}, {FAKE}, 1.0, 8, (1 << 32) - 1, 4, 64", "fewer than 2^32 - 1 rows"),
    ("embedding_i_ij", f"{FAKE}, {FAKE}, {FAKE}, 1.0, 8, 10, 1 << 31, 64", "at most 2^31 - 1 tokens"),
    ("embedding_i_ij", f"{FAKE}, {FAKE}, {FAKE}, 1.0, 8, 10, 4, (1 << 30) + 1", "row length must not exceed"),
    ("embedding_i_ij_reverse", f"{FAKE}, {FAKE}, {FAKE}, None, 1.0, 0.0, 8, 10, 4, 64", "mpEmbeddingReverseScratchBytes"),
    ("embedding_i_ij_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE + 8}, 1.0, 0.0, 8, 10, 4, 64", "16-byte aligned"),
    ("embedding_i_ij_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, 1.0, 0.0, 5, 10, 4, 64", "4 or 8 bytes wide"),
    ("gradient_norm", f"A({FAKE}), L(5), {FAKE}, None, 0.0, 1", "mpGradientNormScratchBytes"),
    ("gradient_norm", f"A({FAKE}), L(5), None, {FAKE}, 0.0, 1", "one aligned double"),
    ("gradient_norm", f"A({FAKE}), L(5), {FAKE + 4}, {FAKE}, 0.0, 1", "one aligned double"),
    ("gradient_norm", f"None, L(5), {FAKE}, {FAKE}, 0.0, 1", "must not be NULL"),
    ("gradient_norm", f"A(None), L(5), {FAKE}, {FAKE}, 0.0, 1", "address is NULL"),
    ("gradient_norm", f"A({FAKE}), L(1 << 60), {FAKE}, {FAKE}, 0.0, 1", "out of range"),
    ("gradient_scale", f"A({FAKE}), None, L(5), {FAKE}, 1.0, 1", "must not be NULL"),
    ("gradient_scale", f"A({FAKE}), A(None), L(5), {FAKE}, 1.0, 1", "address is NULL"),
    ("gradient_scale", f"A({FAKE}), A({FAKE}), L(5), {FAKE}, -1.0, 1", "must not be negative"),
    ("gradient_clip", f"A({FAKE}), A({FAKE}), L(5), {FAKE}, {FAKE}, float('nan'), 1", "must not be negative"),
    ("gradient_clip", f"A({FAKE}, {FAKE}), A({FAKE}, {FAKE}), L(5, 5), {FAKE}, {FAKE}, 1.0, 2", "overlaps another"),
    ("gradient_clip", f"A({FAKE}, {FAKE + 64}), A({FAKE + 128}, {FAKE + 144}), L(5, 5), {FAKE}, {FAKE}, 1.0, 2", "overlaps another"),
    ("gradient_clip", f"A({FAKE}, {FAKE + 64}), A({FAKE + 256}, {FAKE + 4}), L(5, 5), {FAKE}, {FAKE}, 1.0, 2", "overlaps another"),
    ("gradient_scale", f"A({FAKE}), A({FAKE + 16}), L(5), {FAKE}, 1.0, 1", "overlaps another"),
    ("gradient_scale", f"A({FAKE + 512}, {FAKE}, {FAKE + 100}), A({FAKE + 512}, {FAKE}, {FAKE + 100}), L(5, 26, 5), {FAKE}, 1.0, 3", "overlaps another"),
]


@pytest.mark.parametrize("stem,args,message", CASES)
def test_a_call_that_cannot_be_right_is_refused(stem, args, message):
    code = textwrap.dedent(f"""
        import ctypes
        from metaphor_amd import ffi
        kernels, _ = ffi.load()
        A = lambda *p: (ctypes.c_void_p * len(p))(*p)
        L = lambda *p: (ctypes.c_ulong * len(p))(*p)
        ffi.invoke(kernels.{stem}, ffi.R32, {args}, ffi.StreamContext.from_handle(None))
        print("accepted")
    """)
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ffi.ROOT, timeout=120)
    assert res.returncode != 0 and "accepted" not in res.stdout, res.stdout
    assert message in res.stderr, res.stderr


def test_workspace_sizes():
    kernels, _ = ffi.load()
    for key, wide in ((ffi.R16, 4), (ffi.R32, 4), (ffi.R64, 8)):
        # the places and keys of the sort twice over and two partial rows at least
        for v, m, n in ((10, 1, 1), (50257, 8192, 1024), (151936, 100000, 33)):
            assert kernels.mpEmbeddingReverseScratchBytes(key, v, m, n) >= 16 * m + 2 * n * wide
        assert kernels.mpEmbeddingReverseScratchBytes(key, 10, 0, 8) >= 0
        for count in (1, 96, 97, 1000):
            assert kernels.mpGradientNormScratchBytes(key, count) % 8 == 0 and kernels.mpGradientNormScratchBytes(key, count) >= 8
        assert kernels.mpGradientNormScratchBytes(key, 0) == 0


MANY = [
    # 2^24 workgroups of 256 threads are 2^32 threads, more than a launch takes
    ("gradient_scale", f"A({FAKE}), A({FAKE}), L(1 << 36), {FAKE}, 1.0, 1", "too many elements"),
    ("gradient_scale", f"A({FAKE}, {FAKE + (1 << 44)}), A({FAKE}, {FAKE + (1 << 44)}), L(1 << 35, 1 << 35), {FAKE}, 1.0, 2", "too many elements"),
    ("gradient_clip", f"A({FAKE}), A({FAKE + (1 << 44)}), L(1 << 36), {FAKE}, {FAKE}, 1.0, 1", "too many elements"),
    # every refusal comes before the first launch, which without a GPU ends the process with another message
    ("embedding_i_ij", f"{FAKE}, {FAKE}, {FAKE}, 1.0, 8, 10, (1 << 31) - 1, 1 << 20", "too many rows"),
    ("embedding_i_ij_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, 1.0, 0.0, 8, (1 << 32) - 2, 9000, 1 << 20", "too many rows"),
    ("embedding_i_ij_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, 1.0, 0.0, 8, (1 << 32) - 2, 300, 1 << 20", "too many rows"),
    ("embedding_i_ij_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, 1.0, 0.0, 8, (1 << 32) - 2, 20, 1 << 20", "too many rows"),
    ("embedding_i_ij_reverse", f"{FAKE}, {FAKE}, {FAKE}, {FAKE}, 1.0, 1.0, 8, 10, (1 << 31) - 1, 1 << 30", "too many rows"),
]


@pytest.mark.parametrize("stem,args,message", MANY)
def test_more_than_a_launch_takes_is_refused_before_the_first_one(stem, args, message):
    test_a_call_that_cannot_be_right_is_refused(stem, args, message)
