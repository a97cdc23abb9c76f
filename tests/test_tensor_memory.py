"""Tensor memory is given back before a CTA waits for the other CTAs of its cluster.

An SM has 512 columns, and nothing keeps CTAs off it that together want more: an allocation then waits until a neighbour
frees some.  A CTA that holds columns while it waits for a peer, which waits for columns on another SM, closes a circle
with a cluster that stands the other way round, and none of these waits ends.  Kernels launched in clusters of independent
MMA streams (cta_group::1) therefore free theirs first.  (Pair kernels take all 512 columns of both SMs, and the shared
memory of one leaves no room for a second on an SM.)"""
import os
import re

import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocm_dev_b200", "csrc")


def kernels(file):
    """Bodies of a file's kernels without comments, by name."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, file)).read())
    parts = re.split(r"\b__global__\b", text)[1:]
    return {re.search(r"(\w+_kernel)\s*\(", p).group(1): p for p in parts}


@pytest.mark.parametrize("file,kernel", [("fp4_gemm.cu", "split_kernel"), ("skinny_gemm.cu", "skinny_gemm_kernel"),
                                         ("sparse_gemm.cu", "sparse_gemm_kernel")])
def test_columns_are_freed_before_peers_are_waited_for(file, kernel):
    body = kernels(file)[kernel]
    held = body[body.index("tmem_alloc("):]
    first_wait = held.index("cluster_wait_acquire(")
    assert "tmem_dealloc(" in held[:first_wait], "waits for its peers with columns allocated"
    assert body.count("tmem_dealloc(") == 1


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["mxfp4", "nvfp4"])
def test_clusters_of_several_streams_share_the_columns(cuda_device, form):
    """Short products, whose CTAs are small enough for three and more to an SM and cut K over clusters, on four streams at
    once, together with products by CTA pairs that want whole SMs."""
    import rocm_dev_b200 as R
    g = torch.Generator(device=cuda_device).manual_seed(0)
    hold = lambda r, k: R.quantize_fp4(torch.randn((r, k), generator=g, device=cuda_device).bfloat16(), form)  # noqa: E731
    work = []
    for M, N, K in ((16, 2048, 512), (16, 2048, 2048), (7, 4096, 1024), (32, 1024, 2048)):
        work.append((R.skinny_gemm_fp4, hold(M, K), hold(N, K)))
    work.append((lambda a, b: R.dense_gemm_fp4(a, b, tiling=2), hold(512, 768), hold(4096, 768)))
    want = [f(a, b) for f, a, b in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in work]
    graphs, outs = [], []
    for (f, a, b), s in zip(work, streams):             # graphs: launches that follow one another as fast as they can
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append([f(a, b) for _ in range(20)])
        graphs.append(graph)
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert R.lib().rdb_device_status() == 0
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
