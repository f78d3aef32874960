"""The serving loop over a paged cache (paged_serving.py).  CPU: requests, pages and steps with the paged operators restated by
the oracle, token for token against LlamaDecoder.generate.  GPU: the HIP operators in the loop, eager and recorded, every chosen
token against the logits that the float32 CPU model gives the same text."""

import threading

import pytest
import torch

import llama_arch as la
from oracle import cpu_baseline, ops_ref
from paged_serving import PagedServer
from test_harness import tiny_config


class CpuOps:
    rms_norm = staticmethod(cpu_baseline.rms_norm_cpu)
    rot_embed = staticmethod(cpu_baseline.rot_embed_cpu)
    flash_attention_decode = staticmethod(cpu_baseline.attention_cpu)

    @staticmethod
    def norm_rot_embed(q, k, wq, wk, freq, eps):
        return tuple(torch.stack([torch.from_numpy(ops_ref.norm_rot_ref(row, w, freq, eps)) for row in x]).to(x.dtype)
                     for x, w in ((q, wq), (k, wk)))

    @staticmethod
    def rot_embed_append_paged(qkv, freq, k_pages, v_pages, table, q_offsets, kv_lens, n_head, wq, wk, eps):
        rows, page, KVH, HD = qkv.shape[0], *k_pages.shape[1:]
        q, k, v = (t.reshape(rows, -1, HD) for t in qkv.split([n_head * HD, KVH * HD, KVH * HD], dim=-1))
        out = torch.zeros_like(q)
        for row, b, pos in ops_ref.paged_rows_ref(rows, q_offsets.tolist(), kv_lens.tolist()):
            at = table[b, pos // page], pos % page
            one = slice(row, row + 1)
            out[row] = torch.from_numpy(ops_ref.norm_rot_ref(q[one], wq, freq[pos:pos + 1], eps))[0]
            k_pages[at] = torch.from_numpy(ops_ref.norm_rot_ref(k[one], wk, freq[pos:pos + 1], eps))[0].to(k_pages.dtype)
            v_pages[at] = v[row]
        return out

    @staticmethod
    def flash_attention_paged(q, k_pages, v_pages, table, q_offsets, kv_lens, max_new=0):
        assert max_new == 0 or max_new >= int((q_offsets[1:] - q_offsets[:-1]).max())
        return torch.from_numpy(ops_ref.attention_paged_ref(q, k_pages, v_pages, table.numpy(), q_offsets.tolist(),
                                                            kv_lens.tolist())).to(q.dtype)


def model(cfg, ops, device, dtype, seed=42):
    """Layers that outweigh the embedding of the last token: without, the answers mostly repeat it."""
    m = la.LlamaDecoder(cfg, ops, device, dtype=dtype, seed=seed)
    for L in m.layers:
        for name in ("c_attn", "c_proj", "c_fc", "c_fc2", "mlp_proj"):
            L[name] *= 4
    return m


PROMPTS = [la.random_prompts(1, n, 900, n)[0] for n in (9, 1, 30, 17, 2, 12, 33)]


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("pages,sequences,rows", [(40, 7, 512), (40, 3, 8), (7, 7, 20), (12, 2, 2)])
def test_answers_are_those_of_one_sequence_at_a_time(pages, sequences, rows, qk_norm):
    m = model(tiny_config(qk_norm=qk_norm), CpuOps, "cpu", torch.float32)
    want = [m.generate([p], 6, ignore_eos=True)[0] for p in PROMPTS]
    server = PagedServer(m, pages, page_size=8, max_sequences=sequences, max_rows=rows)
    for _ in range(2):      # the second time in pages that hold the first one's keys and values
        assert server.generate(PROMPTS, 6, ignore_eos=True) == want
        assert sorted(server.free) == list(range(pages))


def test_stop_tokens_echo_and_limits():
    m = model(tiny_config(), CpuOps, "cpu", torch.float32)
    free = PagedServer(m, 40, page_size=8).generate(PROMPTS[:3], 6, ignore_eos=True)
    m.tokenizer.stop_tokens = (free[0][2],)
    server = PagedServer(m, 40, page_size=8)
    assert server.generate(PROMPTS[:3], 6) == [m.generate([p], 6)[0] for p in PROMPTS[:3]]
    assert server.generate(PROMPTS[:1], 6)[0] == free[0][:2]
    assert server.generate(PROMPTS[:1], 2, echo=True)[0] == PROMPTS[0] + free[0][:2]
    assert server.generate(PROMPTS[:2], 0) == [[], []] and server.generate([], 5) == []
    longest = la.random_prompts(1, m.config.block_size - 2, 900, 3)[0]      # the text ends with the model's positions
    assert len(server.generate([longest], 9, ignore_eos=True)[0]) == 2


def test_refused_requests_leave_the_pages_free():
    m = model(tiny_config(), CpuOps, "cpu", torch.float32)
    server = PagedServer(m, 4, page_size=8)
    for prompts, error in (([[]], ValueError), ([[5] * 65], ValueError), ([[1000]], IndexError), ([[-1]], IndexError),
                           ([[5], [5] * 30], ValueError)):
        with pytest.raises(error):
            server.generate(prompts, 6)
        assert len(server.free) == 4
    for kw in (dict(page_size=12), dict(page_size=4), dict(pages=0), dict(max_sequences=0), dict(max_sequences=9, max_rows=8)):
        with pytest.raises(ValueError):
            PagedServer(m, **{"pages": 4, **kw})
    m.ops = type("Failing", (CpuOps,), {"flash_attention_paged": staticmethod(lambda *a: 1 / 0)})
    with pytest.raises(ZeroDivisionError):
        server.generate([[5]], 6)
    assert len(server.free) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("n_head,n_kv_head,hd", [(4, 2, 64), (8, 2, 128)])
def test_hip_operators_in_the_loop_choose_the_cpu_models_tokens(gpu, n_head, n_kv_head, hd, qk_norm):
    """A chosen token's float32 logit lies within twice the logits' error of the best: 0.04 of their scale each, which is what
    the harness's tests allow the bf16 model."""
    from custom_kernels import custom_kernels_extension as cke

    cfg = tiny_config(n_head=n_head, n_kv_head=n_kv_head, n_embd=n_head * hd, qk_norm=qk_norm)
    dut = model(cfg, cke, gpu, torch.bfloat16, seed=7)
    ref = la.LlamaDecoder(cfg, CpuOps, "cpu", dtype=torch.float32, weights_from=dut)
    for kw in (dict(pages=64, max_rows=512), dict(pages=64, max_rows=24, max_sequences=20, graphs=False),
               dict(pages=24, max_rows=40, max_sequences=5)):
        print(f"paged serving {n_head}/{n_kv_head} x {hd} norms {qk_norm} {kw}", flush=True)
        server = PagedServer(dut, page_size=8, **kw)
        for _ in range(2):
            answers = server.generate(PROMPTS, 8, ignore_eos=True)
            for prompt, answer in zip(PROMPTS, answers):
                assert len(answer) == 8
                text = torch.tensor([prompt + answer])
                with torch.inference_mode():
                    for i, token in enumerate(answer):
                        logits = ref.forward(text[:, :len(prompt) + i])[0, -1]
                        assert logits[token] >= logits.max() - 2 * 0.04 * logits.abs().max(), (len(prompt), i)
        assert server.steps["mixed"] > 0 and (server.graphs is None or server.steps["generating"] > 0)
        assert server.graphs is None or all(entry[0] is not None for entry in server.graphs.values())


@pytest.mark.gpu
def test_model_with_head_norms_matches_cpu_logits(gpu):
    """norm_rot_embed in the dense path: prompt pass and single tokens, bounds as for the model without norms."""
    from custom_kernels import custom_kernels_extension as cke

    for rows in (3, 7):
        cfg = tiny_config(n_head=8, n_kv_head=2, n_embd=512, qk_norm=True, max_gen_batch_size=rows)
        dut = model(cfg, cke, gpu, torch.bfloat16, seed=7)
        ref = la.LlamaDecoder(cfg, CpuOps, "cpu", dtype=torch.float32, weights_from=dut)
        ids = torch.tensor(la.random_prompts(rows, 20, 900, 11))
        with torch.inference_mode():
            for lo, hi in ((0, 18), (18, 19), (19, 20)):
                a = ref.forward(ids[:, lo:hi], start_pos=lo)
                b = dut.forward(ids[:, lo:hi].to(gpu), start_pos=lo).cpu()
                assert (a - b).abs().max() <= 0.04 * a.abs().max(), (rows, lo)
        with pytest.raises(NotImplementedError):
            dut.generate_graphed(ids.tolist(), 4)
        assert [len(t) for t in dut.generate(ids.tolist(), 4, ignore_eos=True)] == [4] * rows


def test_recorded_steps_go_with_the_model_they_were_recorded_of():
    m = model(tiny_config(qk_norm=True), CpuOps, "cpu", torch.float32)
    server = PagedServer(m, 4, page_size=8)
    server.graphs = {}
    server.generate([], 1)

    def changes():
        m.decode_linear_rows = 8
        yield
        m.layers[1]["c_proj"] = m.layers[1]["c_proj"].clone()
        yield
        m.layers[0]["k_norm"] = m.layers[0]["k_norm"].clone()
        yield
        m.ln_f = m.ln_f.clone()
        yield
        m.wte = torch.zeros(m.wte.shape[0], m.wte.shape[1] + 8)[:, :-8].copy_(m.wte)
        yield
        m.ops = type("Others", (CpuOps,), {})
        yield

    for _ in changes():
        server.graphs[4] = (None, None, None)
        server.generate([], 1)
        assert not server.graphs
        server.graphs[4] = (None, None, None)
        server.generate([], 1)      # nothing is another: recorded steps stay
        assert server.graphs


@pytest.mark.gpu
def test_a_server_answers_with_the_models_present_weights(gpu):
    """The steps it had recorded read the weights that were replaced (kept alive here)."""
    from custom_kernels import custom_kernels_extension as cke

    cfg = tiny_config(n_head=4, n_kv_head=2, n_embd=256)
    dut, other = (model(cfg, cke, gpu, torch.bfloat16, seed=s) for s in (7, 8))
    server = PagedServer(dut, 64, page_size=8)
    first = server.generate(PROMPTS, 8, ignore_eos=True)
    kept = dut.wte, dut.layers
    dut.wte, dut.layers = other.wte, other.layers
    want = PagedServer(other, 64, page_size=8).generate(PROMPTS, 8, ignore_eos=True)
    print("weights replaced under a server with recorded steps", flush=True)
    assert server.generate(PROMPTS, 8, ignore_eos=True) == want != first
    dut.wte, dut.layers = kept
    dut.set_decode_linear_rows(0)
    want = PagedServer(dut, 64, page_size=8).generate(PROMPTS, 8, ignore_eos=True)
    assert server.generate(PROMPTS, 8, ignore_eos=True) == want


def chosen_tokens_are_near_the_best(ref, prompts, answers, length):
    """The bound of test_hip_operators_in_the_loop_choose_the_cpu_models_tokens, with one pass over each text."""
    for prompt, answer in zip(prompts, answers):
        assert len(answer) == length
        for i, token in enumerate(answer):
            with torch.inference_mode():
                logits = ref.forward(torch.tensor([prompt + answer[:i]]))[0, -1]
            assert logits[token] >= logits.max() - 2 * 0.04 * logits.abs().max(), (len(prompt), i)


def transposed(w):
    return w.t().contiguous().t()


@pytest.mark.gpu
@pytest.mark.parametrize("what,sequences", [("width", 7), ("width", 20), ("transposed", 20)])
def test_generating_steps_of_weights_that_the_streaming_linears_refuse(gpu, what, sequences):
    """Widths that are no multiple of 128, and weights that lie the other way round (which steps of more than 16 rows take
    everywhere else): such a model's generating steps take the linears that its other steps take."""
    from custom_kernels import custom_kernels_extension as cke

    cfg = tiny_config(n_head=3, n_kv_head=1, n_embd=192, hidden_dim=320) if what == "width" else tiny_config()
    dut = model(cfg, cke, gpu, torch.bfloat16, seed=7)
    ref = la.LlamaDecoder(cfg, CpuOps, "cpu", dtype=torch.float32, weights_from=dut)
    for L in dut.layers if what == "transposed" else ():
        for name in ("c_attn", "c_proj", "mlp_proj"):
            L[name] = transposed(L[name])
    prompts = [la.random_prompts(1, 18 if what == "transposed" else 3 + i % 4, 900, i)[0] for i in range(sequences)]
    for graphs in (False, True):
        print(f"{what}, {sequences} sequences, graphs {graphs}", flush=True)
        server = PagedServer(dut, 80, page_size=8, max_sequences=sequences, graphs=graphs)
        chosen_tokens_are_near_the_best(ref, prompts, server.generate(prompts, 4, ignore_eos=True), 4)
        assert server.graphs is None or [entry[0] is not None for entry in server.graphs.values()] == [True]


def test_calls_from_several_threads_take_turns():
    """The second call comes while the first holds every page and has a step half done."""
    m = model(tiny_config(), CpuOps, "cpu", torch.float32)
    want = [m.generate([p], 6, ignore_eos=True)[0] for p in PROMPTS[:2]]
    server, answers, errors, began = PagedServer(m, 2, page_size=8), {}, [], threading.Event()

    def call(i):
        try:
            answers[i] = server.generate([PROMPTS[i]], 6, ignore_eos=True)[0]
        except Exception as e:      # noqa: BLE001 (shown below)
            errors.append(e)

    threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]

    def interrupted(*a):
        if not began.is_set():
            began.set()
            threads[1].start()
            threads[1].join(0.5)      # it is through only if it did not wait for this call
        return CpuOps.flash_attention_paged(*a)

    m.ops = type("Interrupted", (CpuOps,), {"flash_attention_paged": staticmethod(interrupted)})
    threads[0].start()
    for t in threads:
        began.wait(10)
        t.join(10)
    assert not errors and answers == dict(enumerate(want)) and sorted(server.free) == [0, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("requests,sequences,qk_norm", [(20, 20, False), (23, 20, True), (64, 64, False), (64, 64, True), (70, 64, False)])
def test_generating_steps_of_many_sequences(gpu, requests, sequences, qk_norm, graphs):
    """Steps of 17 to 64 rows have linears of their own; 20 sequences make a step that is no power of two."""
    from custom_kernels import custom_kernels_extension as cke

    cfg = tiny_config(n_head=4, n_kv_head=2, n_embd=256, qk_norm=qk_norm)
    dut = model(cfg, cke, gpu, torch.bfloat16, seed=7)
    ref = la.LlamaDecoder(cfg, CpuOps, "cpu", dtype=torch.float32, weights_from=dut)
    prompts = [la.random_prompts(1, 1 + 5 * i % 23, 900, i)[0] for i in range(requests)]
    print(f"{requests} requests, {sequences} at once, norms {qk_norm}, graphs {graphs}", flush=True)
    server = PagedServer(dut, 64 * 4, page_size=8, max_sequences=sequences, max_rows=512, graphs=graphs)
    chosen_tokens_are_near_the_best(ref, prompts, server.generate(prompts, 4, ignore_eos=True), 4)
    assert not graphs or sequences in server.graphs and all(entry[0] is not None for entry in server.graphs.values())
