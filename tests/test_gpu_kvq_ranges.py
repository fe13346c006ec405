"""Quantised caches: how keys are cut into ranges over sequences of different lengths and joined
again, at the counts where the joining takes another way."""
import pytest
import torch
from test_gpu_kvq import check_gqa, check_paged, make_gqa, make_paged, run_gqa, run_paged

pytestmark = pytest.mark.gpu


# Ranges of a lone sequence have 512 keys at least: 1, 2, 3, 4, 5, 17 and 33 of them, and a last
# one of a single key.
@pytest.mark.parametrize("past", [511, 512, 1024, 1600, 2048, 8200, 16640])
def test_ranges_of_a_token(ortmi, past):
    run_gqa(ortmi, S=1, past=past, KV=1, hd=64)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [96, 128])
def test_ranges_of_a_token_types(ortmi, dtype, hd):
    run_gqa(ortmi, S=3, past=2500, hd=hd, dtype=dtype, code="int4")


def test_ragged_ranges(ortmi):
    """Sequences of one range, of several and of none beside each other."""
    run_gqa(ortmi, B=6, S=1, past=3000, lens=[1, 3001, 512, 513, 2000, 0])
    run_gqa(ortmi, B=5, S=4, past=2000, lens=[2004, 3, 0, 1024, 700], H=3, KV=1)


@pytest.mark.parametrize("B", [63, 64, 65, 130])
def test_many_sequences(ortmi, B):
    """More of them than a wave has lanes."""
    run_gqa(ortmi, B=B, S=1, past=700, KV=1, H=2, hd=64, code="fp8",
            lens=[(37 * i) % 702 for i in range(B)])


@pytest.mark.parametrize("S,past", [(33, 4000), (70, 9000)])
def test_ranges_of_a_prompt(ortmi, S, past):
    run_gqa(ortmi, S=S, past=past, KV=1, H=4, hd=64, code="fp8")


def test_padded_prompt_over_several_ranges(ortmi):
    run_gqa(ortmi, B=3, S=40, past=1500, lens=[1540, 20, 800])


# Ranges of 256 keys: 1, 2, 3, 5, 17, 33 for one prompt tile.
@pytest.mark.parametrize("past", [200, 300, 700, 1100, 4200, 8300])
def test_ranges_of_a_page_tile(ortmi, past):
    run_paged(ortmi, past=(past,), new=(9,), KV=2, H=4, code="int4")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [96, 128])
def test_ranges_of_pages_types(ortmi, dtype, hd):
    run_paged(ortmi, past=(1900, 2100, 5), new=(20, 1, 3), hd=hd, dtype=dtype, sink=True)


@pytest.mark.parametrize("blk", [16, 48, 80, 112, 1040])
def test_page_sizes_over_ranges(ortmi, blk):
    """Sizes that are not powers of two, across the ends of ranges."""
    run_paged(ortmi, past=(1500, 600, 40), new=(1, 30, 70), blk=blk)


def test_sequences_by_the_hundred(ortmi):
    """Token and prompt sequences and empty ones, three times the lanes of a wave."""
    new = [(0, 1, 1, 9, 2)[i % 5] for i in range(190)]
    past = [(97 * i) % 900 for i in range(190)]
    run_paged(ortmi, past=tuple(past), new=tuple(new), H=4, KV=1, hd=64)


def test_all_sequences_empty(ortmi):
    args, t = make_paged(past=(30, 9), new=(0, 0), extra=3)
    ws = torch.zeros(ortmi.load_kernels().ortmi_paged_attention_quantized_workspace_size(
        3, 2, 4, 2, 64, 48), dtype=torch.uint8, device="cuda")
    before = args["key_cache"].clone()
    ortmi.paged_attention_quantized(**{**args, "max_context": 48}, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(args["key_cache"].view(torch.uint8), before.view(torch.uint8))


def test_two_graphs_on_one_workspace(ortmi):
    """Captured calls that share a workspace, replayed in turn with eager work between."""
    made = [make_gqa(S=1, past=p, hd=128, KV=2, H=8, seed=i) for i, p in enumerate((1800, 4100))]
    lib = ortmi.load_kernels()
    need = max(lib.ortmi_group_query_attention_quantized_workspace_size(1, 1, 8, 2, 128, n)
               for n in (1801, 4101))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    want = [ortmi.group_query_attention_quantized(**a)[0].clone() for a, _ in made]
    graphs, outs = [], []
    for a, _ in made:
        ortmi.group_query_attention_quantized(**a, workspace=ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ortmi.group_query_attention_quantized(**a, workspace=ws)[0])
        graphs.append(graph)
    for i in (0, 1, 1, 0, 1, 0):
        outs[i].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i])
        eager = ortmi.group_query_attention_quantized(**made[1 - i][0])
        torch.cuda.synchronize()
        check_gqa(ortmi, eager, made[1 - i][1])


def test_same_result_every_time(ortmi):
    """Ranges are joined in one order: outputs do not change from call to call."""
    args, t = make_paged(past=(3000, 1200, 50), new=(1, 40, 2), H=8, KV=2, hd=128)
    first = ortmi.paged_attention_quantized(**args).clone()
    for _ in range(5):
        assert torch.equal(ortmi.paged_attention_quantized(**args), first)
    check_paged(first, args, t)


def test_the_stream_of_the_call(ortmi):
    """stream=: run there, in order with its other work, whatever the current stream does."""
    side = torch.cuda.Stream()
    args, t = make_gqa(S=1, past=3000, hd=128)
    pages, pt = make_paged(past=(2500, 700), new=(1, 30), hd=128)
    logits = torch.randn((3, 5000), device="cuda")
    u = torch.rand(3, device="cuda")
    ids = ortmi.sample_rows(logits, u, top_k=40)[0]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # the calls wait behind this
        fill = [args["query"].clone(), pages["query"].clone(), logits.clone()]
    args["query"], pages["query"] = fill[:2]
    out = ortmi.group_query_attention_quantized(**args, stream=side.cuda_stream)
    paged = ortmi.paged_attention_quantized(**pages, stream=side.cuda_stream)
    drawn = ortmi.sample_rows(fill[2], u, top_k=40, stream=side.cuda_stream)[0]
    junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]
    side.synchronize()
    torch.cuda.synchronize()
    check_gqa(ortmi, out, t)
    check_paged(paged, pages, pt)
    assert torch.equal(drawn, ids)
    del junk


def test_prompts_by_the_hundred(ortmi):
    """More sequences with prompt tiles than the GPU has CUs."""
    new = [5 + i % 4 for i in range(300)]
    past = [(53 * i) % 400 for i in range(300)]
    run_paged(ortmi, past=tuple(past), new=tuple(new), H=4, KV=1, hd=64, code="int4")


@pytest.mark.parametrize("new", [(1, 1, 1), (20, 1, 40)])
def test_shared_prefix(ortmi, new):
    """Sequences that read the same first blocks."""
    args, t = make_paged(past=(70, 64, 90), new=new, hd=128, H=8, blk=16)
    t["bt"][1:, :4] = t["bt"][0, :4]
    args["block_table"].copy_(t["bt"])
    out = ortmi.paged_attention_quantized(**args)
    torch.cuda.synchronize()
    check_paged(out, args, t)
