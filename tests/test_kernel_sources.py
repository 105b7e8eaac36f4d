"""What the kernels' sources must hold to, read as text.  A kernel that is launched while the one in front still runs may read what
that one writes after its wait only, and then through a pointer that may have changed: a const __restrict__ parameter counts
as unchanged for the whole kernel, from ahead of the wait on."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "airun_b200", "csrc")
SOURCES = {os.path.basename(p): re.sub(r"//[^\n]*", "", open(p).read()) for p in sorted(glob.glob(os.path.join(CSRC, "*.cu*")))}


def test_work_lists_are_read_fresh():
    """The lists of csrc/attention_plan.cu: tiles, rows of single tokens and their numbers."""
    readers = 0
    for name, text in SOURCES.items():
        if name == "attention_plan.cu":
            continue
        assert not re.search(r"__restrict__\s+(tiles|n_tiles_dev|n_rows_dev)\b", text), name
        for use in re.finditer(r"\*\s*(?:x\.)?(n_tiles_dev|n_rows_dev)\b|\b(?:x\.rows|tiles)\[", text):
            before = text[max(0, use.start() - 30):use.start()]
            assert re.search(r"(const )?(int|int32_t|int4|void)\s*$", before), (name, text[use.start() - 60:use.end() + 20])
        readers += len(re.findall(r"load_fresh\(", text))
    assert readers >= 8


# what no kernel of a step writes: weights and constants of the model, the batch's layout and lists that are copied to the device
# ahead of the step, sampling parameters
UNWRITTEN = set("""W alpha b bias c1 c2 s1 s2 correction dist_a dist_b group_param head_c head_decay inv_freq k_bias q_bias v_bias k_norm_w
q_norm_w k_w q_w mu norm_w sink table vec w w2 w_post w_post2 w_pre wkv wq y_bias
block_table context_lens cu_tokens positions req_of_token rows state_slots pairs temperature uniform""".split())
# results that their kernel does not read, or reads only what it has written itself
WRITTEN_ONLY = set("""C cast coef counts cq dst err out out2 out_flags out_ids out_vals partial pool q_out qlat qn row_of rows seg tiles xs""".split())


def test_what_a_step_writes_is_not_read_as_unchanging():
    """Every __restrict__ parameter in front of a wait is one that nothing writes, or one that is not read."""
    seen = 0
    for name, text in SOURCES.items():
        for m in re.finditer(r"(const\s+)?\w+\s*\*\s*__restrict__\s+(\w+)", text):
            seen += 1
            assert m.group(2) in (UNWRITTEN if m.group(1) else WRITTEN_ONLY), (name, m.group(0))
        # a cached load by name counts as unchanging too
        for m in re.finditer(r"__ldg\((?:reinterpret_cast<const \w+\*>\()?([\w.]+)", text):
            assert m.group(1).split(".")[-1] in UNWRITTEN | {"bt", "wr", "src"}, (name, m.group(0))
    assert seen > 100
    head = SOURCES["linear_attention.cu"].split("gla_segment_kernel(")[1].split("{")[0]
    assert re.search(r"float\*\s+out\b", head)                       # this one adds to what is there


def test_kernels_wait_before_they_end_and_trigger_first():
    """A kernel that is launched early and never waits would let the kernel behind it start over unfinished work.  Every kernel is looked at, however it is launched
    (by name, through a variable or a macro, in clusters), but for those launched without the attribute."""
    seen = set()
    for name, text in SOURCES.items():
        plain = set(re.findall(r"\b(\w+)(?:<[^<>;()]*>)?\s*<<<", text))
        for at in re.finditer(r"__global__\s*(?:__launch_bounds__\([^)]*\))?\s*void\s+(\w+)\s*\(", text):
            if at.group(1) in plain:
                continue
            end = text.find("__global__", at.end())
            body = text[at.end():end if end > 0 else len(text)]
            assert "pdl_wait()" in body and "pdl_trigger()" in body and body.index("pdl_trigger()") < body.index("pdl_wait()"), (name, at.group(1))
            seen.add(at.group(1))
        assert len(re.findall("__global__", text)) == len(re.findall(r"__global__\s*(?:__launch_bounds__\([^)]*\))?\s*void\s+\w+\s*\(", text)), name
        launched = set(re.findall(r"\bairun_launch\w*\(\(*(\w+?)(?:<|,)", text))
        assert launched <= seen | {"kern", "KERNEL", "kernel"}, (name, launched - seen)
    assert {"gemm_pair_kernel", "gemm_tcgen05_kernel", "gemm_rows_kernel", "delta_chunk_kernel"} <= seen


def test_bounded_waits_come_behind_the_wait_for_the_kernel_in_front():
    """A wait on a barrier gives up after two seconds, but the kernel in front may run for longer: a warp that stood at a barrier meanwhile, for operands that another
    warp asks for behind its pdl_wait(), would report a wait that has run out.  Every warp passes pdl_wait() first, most once and for all roles."""
    seen = set()
    for name, text in SOURCES.items():
        for at in re.finditer(r"__global__[^;{]*?\bvoid\s+(\w+)\s*\(", text):
            body = text[at.end():text.find("\n}\n", at.end())]
            if not re.search(r"\bmbar_(try_)?wait", body):
                continue
            seen.add(at.group(1))
            if at.group(1) == "attn_decode_kernel":                # one flow for all threads, which waits early or behind the first loads
                front = body[:body.rindex("pdl_wait();")]
            elif at.group(1) == "gemm_f32_parts_kernel":           # the last role, the loads', asks for weights first
                assert "const bool loads = warp == X_SUM_WARPS + X_CUT_WARPS + 1;" in body and "if (FORM != 2 && !loads) pdl_wait();" in body
                front = body[:body.index("!loads) pdl_wait();")]
                role = body[body.index("auto ask = "):]
                assert "mbar_wait" not in role[:role.index("if (FORM != 2) pdl_wait();")]
            else:
                wait = re.search(r"^    pdl_wait\(\);", body, re.M)
                assert wait and body.count("pdl_wait();") == 1, at.group(1)
                front = body[:wait.start()]
            assert not re.search(r"\bmbar_(try_)?wait", front), at.group(1)
    assert {"head_logprobs_kernel", "head_few_kernel", "gemm_f32_parts_kernel", "gemm_pair_kernel", "attn_decode_kernel", "latent_prefill_kernel"} <= seen


def test_instructions_of_pairs_of_ctas_are_wrapped_once():
    """Loads, products and commits of cta_group::2 stand in the header that the kernels share, and nothing of that header is written again beside a kernel."""
    shared = set(re.findall(r"__device__ __forceinline__ \w+ (\w+)\(", SOURCES["tcgen05.cuh"]))
    assert {"tma_load_2d_pair", "umma_bf16_pair", "umma_commit_pair", "umma_bf16", "mbar_init"} <= shared
    for name, text in SOURCES.items():
        if name != "tcgen05.cuh":
            assert not shared & set(re.findall(r"__device__ __forceinline__ \w+ (\w+)\(", text)), name
            assert not re.search(r"(cp\.async\.bulk\.tensor\.2d|tcgen05\.mma|tcgen05\.commit)\.cta_group::2", text), name


def test_kernels_hold_their_tensor_memory_before_others_may_start():
    """A kernel behind may be resident as soon as every block has passed pdl_trigger().  If it could take tensor memory that a block in front still has to ask for, it would
    wait for that block to end, and the block for the memory.  So a kernel takes its own first."""
    seen = set()
    for name, text in SOURCES.items():
        for at in re.finditer(r"__global__[^;{]*?\bvoid\s+(\w+)\s*\(", text):
            body = text[at.end():text.find("\n}\n", at.end())]
            asks = [m.start() for m in re.finditer(r"\btmem_alloc\(|tcgen05\.alloc\.", body)]
            if asks:
                seen.add(at.group(1))
                trigger = body.index("pdl_trigger();")
                if at.group(1) == "gemm_f32_parts_kernel":         # all but 4 KB of the shared memory is its own
                    size = lambda n: int(eval(re.sub(r"[A-Z]\w+", lambda m: str(size(m.group(0))), re.search(rf"#define {n} ([^\n]*)", text).group(1))))      # noqa: E731
                    assert 220 * 1024 <= size("X_SMEM") <= 227 * 1024
                    continue
                assert body.count("pdl_trigger();") == 1 and asks[-1] < trigger and "__syncthreads();" in body[asks[-1]:trigger], at.group(1)
    assert {"head_logprobs_kernel", "head_few_kernel", "gemm_tcgen05_kernel", "gemm_tcgen05_persistent_kernel", "gemm_pair_kernel", "gemm_f32_parts_kernel",
            "attn_prefill_tc_kernel", "attn_prefill_wide_kernel", "latent_prefill_kernel"} == seen
