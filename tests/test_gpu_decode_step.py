"""The attention half and the sampler beside the matrix products that they belong to, as a decode step runs them: embedding ->
q | k | v projection -> q norm and rotation -> k norm, rotation and append to the cache -> paged attention -> output
projection + residual -> lm_head -> sampling, every launch on one stream, captured in a HIP graph and replayed."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from hipengine_amd.kernels.hip_gfx950.attention import kv_cache_q8 as C
from hipengine_amd.kernels.hip_gfx950.attention import paged_attention_q8 as A
from hipengine_amd.kernels.hip_gfx950.attention import qk_norm_rope as R
from hipengine_amd.kernels.hip_gfx950.quant import gguf_embedding as E
from hipengine_amd.kernels.hip_gfx950.quant import gguf_q8_1_gemv as G
from hipengine_amd.kernels.hip_gfx950.sampling import sample_rows as S
from oracle import attention_oracle as AO
from oracle import gguf_oracle as O

pytestmark = pytest.mark.gpu

H, HQ, HK, D, V = 1024, 8, 2, 128, 8192
QKV = (HQ + 2 * HK) * D
PAGE, MAX_KV = 64, 9000


class Weights:
    def __init__(self, dev):
        rng = np.random.default_rng(31)
        self.emb = dev.put(O.random_weight(O.GGML_Q4_K, V, H, seed=1, std=1.0))
        self.qkv = dev.put(O.random_weight(O.GGML_Q4_K, QKV, H, seed=2))
        self.out = dev.put(O.random_weight(O.GGML_Q4_K, H, HQ * D, seed=3))
        self.lm = dev.put(O.random_weight(O.GGML_Q6_K, V, H, seed=4))
        self.q_norm, self.k_norm = (dev.put(rng.uniform(0.5, 1.5, D).astype(np.float32)) for _ in range(2))
        self.freq = dev.put((1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32))

    def free(self, dev):
        dev.free(*vars(self).values())


class State:
    """What a step of a batch reads and writes: its cache, its scratch, its outputs."""

    def __init__(self, dev, lens, seed):
        rng = np.random.default_rng(seed)
        self.dev, self.lens, b = dev, np.array(lens, np.int32), len(lens)
        self.b, self.slots = b, (max(lens) + 40 + PAGE - 1) // PAGE
        self.pages = b * self.slots
        self.table = rng.permutation(self.pages).astype(np.int32).reshape(b, self.slots)
        n = self.pages * PAGE * HK * D
        blocks = self.pages * HK * PAGE // 32
        self.bytes = [rng.integers(1, 256, n).astype(np.uint8) for _ in range(2)]
        self.scales = [rng.uniform(0.005, 0.03, blocks).astype(np.float32) for _ in range(2)]
        self.cache = [dev.put(x) for x in (*self.bytes, *self.scales)]
        self.handle = C.KVCacheQ8(*(x.ptr for x in self.cache), self.pages, PAGE, HK, D)
        self.where = dev.put(self.table)
        self.start, self.kv = dev.put(np.arange(b + 1, dtype=np.int32)), dev.put(self.lens)
        self.ids, self.pos = dev.put(np.zeros(b, np.int64)), dev.put(np.zeros(b, np.int64))
        self.uniform = dev.put(np.zeros(b, np.float32))
        self.temp, self.top_p = dev.put(np.full(b, 0.8, np.float32)), dev.put(np.full(b, 0.95, np.float32))
        self.top_k = dev.put(np.array([50 if i % 2 else 0 for i in range(b)], np.int32))
        self.outs = {"x": b * H * 2, "qkv": b * QKV * 2, "q": b * HQ * D * 2, "att": b * HQ * D * 2, "h": b * H * 2,
                     "logits": b * V * 4, "next": b * 4, "logprob": b * 4}
        self.outs = {k: dev.empty(v) for k, v in self.outs.items()}
        self.att_bytes = A.paged_attention_q8_workspace_bytes(b, b, 1, MAX_KV, HQ, HK, D)
        self.sample_bytes = S.sample_workspace_bytes(b, V)
        assert self.att_bytes > 0                              # (the chunks' join is part of the step)
        self.scratch = [dev.empty(self.att_bytes), dev.empty(self.sample_bytes)]

    def put(self, ids, lens, uniform):
        rt = self.dev.runtime
        for buf, a in ((self.ids, np.asarray(ids, np.int64)), (self.kv, np.asarray(lens, np.int32)),
                       (self.pos, np.asarray(lens, np.int64) - 1), (self.uniform, np.asarray(uniform, np.float32))):
            rt.memcpy(buf.ptr, a.ctypes.data, a.nbytes, 1)

    def reset(self):
        rt = self.dev.runtime
        for buf, a in zip(self.cache, (*self.bytes, *self.scales)):
            rt.memcpy(buf.ptr, a.ctypes.data, a.nbytes, 1)

    def poison(self):
        for x in (*self.outs.values(), *self.scratch):
            self.dev.runtime.memset(x.ptr, 0x5C, x.nbytes)

    def read(self):
        g, o, b = self.dev.get, self.outs, self.b
        return {"q": g(o["q"], np.uint16, (b, HQ, D)).copy(), "att": g(o["att"], np.uint16, (b, HQ, D)).copy(),
                "logits": g(o["logits"], np.uint32, (b, V)).copy(), "next": g(o["next"], np.int32, (b,)).copy(),
                "logprob": g(o["logprob"], np.uint32, (b,)).copy(),
                **{f"cache {i}": g(x, np.uint8, (x.nbytes,)).copy() for i, x in enumerate(self.cache)}}

    def free(self):
        self.dev.free(*self.cache, self.where, self.start, self.kv, self.ids, self.pos, self.uniform, self.temp, self.top_p,
                      self.top_k, *self.outs.values(), *self.scratch)


def step(w, s, stream):
    o, b = s.outs, s.b
    E.gguf_q4_k_embedding_bf16_out(s.ids.ptr, w.emb.ptr, o["x"].ptr, b, H, V, stream=stream)
    G.FUSED[("q4_k", "bf16", "bf16")](o["x"].ptr, w.qkv.ptr, o["qkv"].ptr, b, H, QKV, stream=stream)
    qkv = o["qkv"].ptr
    R.qk_norm_rope(qkv, None, o["q"].ptr, None, b, HQ, 0, D, q_weight_ptr=w.q_norm.ptr, positions_ptr=s.pos.ptr,
                   inv_freq_ptr=w.freq.ptr, rotary_dim=D, q_stride=QKV, stream=stream)
    C.kv_append_q8(s.handle, qkv + HQ * D * 2, qkv + (HQ + HK) * D * 2, s.where.ptr, s.slots, s.start.ptr, s.kv.ptr, b, b, 1,
                   k_weight_ptr=w.k_norm.ptr, inv_freq_ptr=w.freq.ptr, rotary_dim=D, k_stride=QKV, v_stride=QKV, stream=stream)
    A.paged_attention_q8(s.handle, o["q"].ptr, o["att"].ptr, s.where.ptr, s.slots, s.start.ptr, s.kv.ptr, b, b, 1, MAX_KV, HQ,
                         workspace_ptr=s.scratch[0].ptr, workspace_bytes=s.att_bytes, stream=stream)
    G.gguf_gemv_residual("gguf_q4_k", o["att"].ptr, "bf16", w.out.ptr, o["x"].ptr, o["h"].ptr, "bf16", b, HQ * D, H, stream=stream)
    G.FUSED[("q6_k", "bf16", "f32")](o["h"].ptr, w.lm.ptr, o["logits"].ptr, b, H, V, stream=stream)
    S.sample_f32_rows_i32(o["logits"].ptr, s.uniform.ptr, o["next"].ptr, b, V, workspace_ptr=s.scratch[1].ptr,
                          workspace_bytes=s.sample_bytes, temperature_ptr=s.temp.ptr, top_k_ptr=s.top_k.ptr,
                          top_p_ptr=s.top_p.ptr, out_logprobs_ptr=o["logprob"].ptr, stream=stream)


def capture(rt, w, s, stream):
    rt.stream_begin_capture(stream)
    step(w, s, stream)
    graph = rt.stream_end_capture(stream)
    assert graph
    return graph, rt.graph_instantiate(graph)


def inputs(rng, s, steps):
    return [(rng.integers(0, V, s.b), s.lens + i + 1, rng.random(s.b)) for i in range(steps)]


def check_against_statements(s, got):
    """The attention output from the q and the cache that the step left, and the token from its logits."""
    n = PAGE // 32
    cache = [got[f"cache {i}"] for i in range(4)]
    ki, vi = AO.unpack_cache(*(x.reshape(s.pages, HK, n, D * 32) for x in cache[:2]), D)
    ks, vs = (x.view(np.float32).reshape(s.pages, HK, n).astype(np.float64) for x in cache[2:])
    lens = s.dev.get(s.kv, np.int32, (s.b,))
    q, att = AO.from_bits(got["q"], "bf16"), AO.from_bits(got["att"], "bf16")
    want, dv, mag, arg = AO.attention(q, ki, vi, ks, vs, s.table, np.arange(s.b + 1), lens, scale=D ** -0.5)
    from tests.test_gpu_attention import attention_tolerance

    assert (np.abs(att - want) <= attention_tolerance(want, dv, mag, arg, "bf16", lens.max(), D, 127 * vs.max())).all()
    u = s.dev.get(s.uniform, np.float32, (s.b,))
    for i in range(s.b):
        found = AO.sample(got["logits"][i].view(np.float32), float(u[i]), temperature=float(np.float32(0.8)),
                          top_k=50 if i % 2 else 0, top_p=float(np.float32(0.95)), accuracy=2.0 ** -22)
        assert got["next"][i] in found


def same(got, want):
    for name in want:
        assert np.array_equal(got[name], want[name]), name


@pytest.mark.parametrize("lens", [[8900], [0, 31, 700, 4095, 63]])
def test_step_graph_replays_match_eager(dev, lens):
    """Captured cold, then replayed for five tokens of every sequence, with eager steps on a second, equal state between the
    replays: outputs, logits, tokens and every byte of the cache are the eager step's."""
    rt, rng = dev.runtime, np.random.default_rng(len(lens))
    w, s, e = Weights(dev), State(dev, lens, 5), State(dev, lens, 5)
    stream = rt.stream_create()
    graph, run = capture(rt, w, s, stream)
    for i, given in enumerate(inputs(rng, s, 5)):
        e.put(*given)
        step(w, e, 0)
        want = e.read()
        s.put(*given)
        s.poison()
        rt.device_synchronize()
        rt.graph_launch(run, stream)
        rt.stream_synchronize(stream)
        got = s.read()
        same(got, want)
        if i in (0, 4):
            check_against_statements(s, got)
    rt.graph_exec_destroy(run)
    rt.graph_destroy(graph)
    rt.stream_destroy(stream)
    for x in (s, e):
        x.free()
    w.free(dev)


def test_two_graphs_at_once(dev):
    """Two requests with caches and workspaces of their own, replayed on two streams at the same time."""
    rt, rng = dev.runtime, np.random.default_rng(9)
    w = Weights(dev)
    states = [State(dev, [3000, 17, 1200], 6), State(dev, [5000, 4999], 7)]
    streams = [rt.stream_create() for _ in states]
    graphs = [capture(rt, w, s, x) for s, x in zip(states, streams)]
    given = [inputs(rng, s, 4) for s in states]
    want = []
    for s, steps in zip(states, given):
        for g in steps:
            s.put(*g)
            step(w, s, 0)
            dev.sync()
        want.append(s.read())
        s.reset()
        s.poison()
    for i in range(4):
        for s, steps in zip(states, given):
            s.put(*steps[i])
        rt.device_synchronize()
        for (_, run), x in zip(graphs, streams):
            rt.graph_launch(run, x)
        for x in streams:
            rt.stream_synchronize(x)
    for s, each in zip(states, want):
        same(s.read(), each)
    for (graph, run), x in zip(graphs, streams):
        rt.graph_exec_destroy(run)
        rt.graph_destroy(graph)
        rt.stream_destroy(x)
    for s in states:
        s.free()
    w.free(dev)


def test_step_captures_cold_in_a_fresh_process():
    """Nothing of the library has run in the process before the capture."""
    code = ("import sys; sys.path.insert(0, '.')\n"
            "import tests.test_gpu_decode_step as t\n"
            "from tests._device import Device\n"
            "t.test_step_graph_replays_match_eager(Device(), [40, 8000])\n"
            "print('same')\n")
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
    assert done.stdout.strip().endswith("same")
