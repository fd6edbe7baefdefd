"""Attention over the latents of earlier frames, beside the codec graphs.

Several streams are encoded by the synthetic encoder graph. The latents of a
frame are its tokens; one attention layer (random weights) looks at those of
all earlier frames of its stream. The frames that are there go through prompt
attention in one packed pass, which also fills an INT8 cache; the tokens of the
next frame then come one by one, as an entropy decoder gives them, each a step
of norm and rotation, cache write and token attention on every stream, captured
once into a graph and replayed. At the end the same tokens are run as one prompt
on the contexts read back from the cache, and both results compared.

    python examples/latent_attention.py [--config codec_enc_tiny] [--streams 2] [--frames 2] [--tokens 16]

The projection into queries, keys and values is a matrix product on the host.
Needs the built libraries and an MI355X.
"""

from __future__ import annotations

import argparse
import ctypes as C
import pathlib
import sys
import tempfile
import time

import numpy as np

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "mlvc.cpp_amd" / "python"))

import mlvc_hip  # noqa: E402

Q_HEADS, KV_HEADS, DIM, PAGE = 16, 4, 64, 64
ROW, KV_ROW = Q_HEADS * DIM, KV_HEADS * DIM
SCALE, EPS = DIM ** -0.5, 1e-6


class Device:
    """Device memory and one stream through the device C ABI."""

    def __init__(self):
        self.lib = mlvc_hip.device_lib()
        v, size = C.c_void_p, C.c_size_t
        self.lib.mlvc_hip_malloc.argtypes = [C.POINTER(v), size]
        self.lib.mlvc_hip_free.argtypes = [v]
        for fn in (self.lib.mlvc_hip_memcpy_h2d, self.lib.mlvc_hip_memcpy_d2h):
            fn.argtypes = [v, v, size, v]
        self.stream, self.memory = v(), []
        self.check(self.lib.mlvc_hip_stream_create(C.byref(self.stream)))

    def check(self, rc: int) -> None:
        if rc != 0:
            raise mlvc_hip.MlvcError(self.lib.mlvc_hip_last_error().decode())

    def alloc(self, nbytes: int) -> int:
        p = C.c_void_p()
        self.check(self.lib.mlvc_hip_malloc(C.byref(p), max(nbytes, 16)))
        self.memory.append(p)
        return p.value

    def put(self, a: np.ndarray, at: int | None = None) -> int:
        a = np.ascontiguousarray(a)
        at = self.alloc(a.nbytes) if at is None else at
        self.check(self.lib.mlvc_hip_memcpy_h2d(at, a.ctypes.data, a.nbytes, self.stream))
        self.wait()  # pageable memory: it may go once this returns
        return at

    def get(self, at: int, shape, dtype=np.float16) -> np.ndarray:
        a = np.empty(shape, dtype)
        self.check(self.lib.mlvc_hip_memcpy_d2h(a.ctypes.data, at, a.nbytes, self.stream))
        self.wait()
        return a

    def wait(self) -> None:
        self.check(self.lib.mlvc_hip_stream_synchronize(self.stream))

    def close(self) -> None:
        for p in self.memory:
            self.lib.mlvc_hip_free(p)
        self.check(self.lib.mlvc_hip_stream_destroy(self.stream))


def encode(config: str, streams: int, frames: int) -> list[np.ndarray]:
    """Latents of each stream's frames, [frames, tokens, channels]; stream i has i frames fewer (one at least), and the frame to come."""
    out = []
    with tempfile.TemporaryDirectory() as d:
        mlvc_hip.synth_write(config, d, 0)
        bindings, _ = mlvc_hip.synth_bindings(config)
        with mlvc_hip.Backend(d, "hip", device_id=0) as graph:
            graph.load("MLVCEncoder", bindings)
            for stream in range(streams):
                graph.reset_state()
                latents = []
                for frame in range(max(1, frames - stream) + 1):
                    inputs = [np.array([32], np.int32) if t == np.int32 else
                              mlvc_hip.synth_input(config, i, frame, s, seed=stream)
                              for i, (s, t) in enumerate(zip(graph.in_shapes, graph.in_dtypes))]
                    y = graph.run(inputs)[0].view(np.float16)[0]
                    latents.append(y.reshape(y.shape[0], -1).T)
                out.append(np.stack(latents))
    return out


class Layer:
    """One attention layer and the cache of its streams."""

    def __init__(self, dev: Device, channels: int, contexts: list[int], room: int):
        rng = np.random.default_rng(1)
        self.dev = dev
        self.w_in = rng.normal(0, channels ** -0.5, (channels, ROW + 2 * KV_ROW)).astype(np.float32)
        self.norm_q, self.norm_k = (dev.put(rng.normal(1, 0.1, DIM).astype(np.float16)) for _ in range(2))
        freqs, self.rot_scale = mlvc_hip.rope_frequencies(DIM, 10000.0, mlvc_hip.ROPE_BANDS, 4.0, 8160)
        self.freqs = dev.put(freqs)
        # Every stream gets the pages of its context and of the tokens to come.
        pages = [-(-(n + room) // PAGE) for n in contexts]
        order = rng.permutation(sum(pages)).tolist()
        self.table = np.full((len(pages), max(pages)), -1, np.int32)
        for i, n in enumerate(pages):
            self.table[i, :n] = [order.pop() for _ in range(n)]
        self.device_table = dev.put(self.table)
        self.cache = mlvc_hip.KvCache(kind=mlvc_hip.KV_INT8, pages=sum(pages), page_size=PAGE, heads=KV_HEADS, head_dim=DIM)
        values, scales = mlvc_hip.kv_cache_bytes(self.cache)
        self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale = (
            dev.alloc(n) for n in (values, values, scales, scales))

    def project(self, tokens: np.ndarray) -> np.ndarray:
        """Rows of q, k and v side by side."""
        return (tokens.astype(np.float32) @ self.w_in).astype(np.float16)

    def slots(self, stream: int, positions) -> np.ndarray:
        p = np.asarray(positions)
        return (self.table[stream, p // PAGE] * PAGE + p % PAGE).astype(np.int32)

    def rotate_and_keep(self, qkv: int, tokens: int, positions: int, slots: int) -> None:
        """Queries and keys in place, keys and values into the cache."""
        q, k, v, stride = qkv, qkv + 2 * ROW, qkv + 2 * (ROW + KV_ROW), ROW + 2 * KV_ROW
        mlvc_hip.qk_norm_rope(mlvc_hip.QkNormRope(
            tokens=tokens, q_heads=Q_HEADS, k_heads=KV_HEADS, head_dim=DIM, q=q, k=k, q_out=q, k_out=k, q_stride=stride,
            k_stride=stride, q_out_stride=stride, k_out_stride=stride, q_weight=self.norm_q, k_weight=self.norm_k, eps=EPS,
            positions=positions, freqs=self.freqs, rot_dim=DIM, interleaved=0, rot_scale=self.rot_scale), self.dev.stream)
        mlvc_hip.kv_write(self.cache, mlvc_hip.KvRows(tokens=tokens, k=k, v=v, k_stride=stride, v_stride=stride, slots=slots),
                          self.dev.stream)

    def prompt(self, q: int, k: int, v: int, strides, out: int, queries: list[int], keys: list[int]) -> None:
        starts_q, starts_k = (self.dev.put(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)) for n in (queries, keys))
        mlvc_hip.attention_prompt(mlvc_hip.PromptAttention(
            sequences=len(queries), q_heads=Q_HEADS, kv_heads=KV_HEADS, head_dim=DIM, q=q, k=k, v=v, out=out,
            q_stride=strides[0], k_stride=strides[1], v_stride=strides[2], out_stride=ROW, q_starts=starts_q,
            k_starts=starts_k, q_tokens=sum(queries), k_tokens=sum(keys), longest_q=max(queries), causal=1, scale=SCALE),
            self.dev.stream)


def run(config: str = "codec_enc_1920x1088", streams: int = 2, frames: int = 2, steps: int = 16) -> dict:
    latents = encode(config, streams, frames)
    past = [y[:-1].reshape(-1, y.shape[2]) for y in latents]
    contexts = [t.shape[0] for t in past]
    steps = min(steps, latents[0].shape[1])
    dev = Device()
    try:
        layer = Layer(dev, latents[0].shape[2], contexts, steps)
        stride = ROW + 2 * KV_ROW

        # The frames that are there: one packed prompt.
        total = sum(contexts)
        qkv, out = dev.put(layer.project(np.concatenate(past))), dev.alloc(2 * total * ROW)
        positions = dev.put(np.concatenate([np.arange(n, dtype=np.int32) for n in contexts]))
        layer.rotate_and_keep(qkv, total, positions, dev.put(np.concatenate([layer.slots(i, np.arange(n)) for i, n in enumerate(contexts)])))
        layer.prompt(qkv, qkv + 2 * ROW, qkv + 2 * (ROW + KV_ROW), (stride,) * 3, out, contexts, contexts)
        finite = bool(np.isfinite(dev.get(out, (total, ROW))).all())

        # The next frame, token by token: the step's buffers stay, so it is captured once.
        row, step_out = dev.alloc(2 * streams * stride), dev.alloc(2 * streams * ROW)
        at, slots, lengths = (dev.alloc(4 * streams) for _ in range(3))
        attend = mlvc_hip.TokenAttention(
            cache=C.pointer(layer.cache), streams=streams, q_heads=Q_HEADS, q=row, out=step_out, q_stride=stride,
            out_stride=ROW, table=layer.device_table, table_stride=layer.table.shape[1], lengths=lengths,
            longest=max(contexts) + steps, scale=SCALE)
        attend.workspace_bytes = mlvc_hip.attention_token_workspace_bytes(attend)
        attend.workspace = dev.alloc(attend.workspace_bytes)
        graph = C.c_void_p()
        dev.check(dev.lib.mlvc_hip_capture_begin(dev.stream))
        layer.rotate_and_keep(row, streams, at, slots)
        mlvc_hip.attention_token(attend, dev.stream)
        dev.check(dev.lib.mlvc_hip_capture_end(dev.stream, C.byref(graph)))
        by_token, rotated, spent = [], [], 0.0
        for step in range(steps):
            dev.put(layer.project(np.stack([y[-1, step] for y in latents])), row)
            dev.put(np.array([n + step for n in contexts], np.int32), at)
            dev.put(np.array([layer.slots(i, n + step) for i, n in enumerate(contexts)], np.int32), slots)
            dev.put(np.array([n + step + 1 for n in contexts], np.int32), lengths)
            began = time.perf_counter()
            dev.check(dev.lib.mlvc_hip_graph_launch(graph, dev.stream))
            dev.wait()
            spent += time.perf_counter() - began
            by_token.append(dev.get(step_out, (streams, ROW)))
            rotated.append(dev.get(row, (streams, stride))[:, :ROW])
        dev.check(dev.lib.mlvc_hip_graph_destroy(graph))

        # The same tokens as one prompt on the contexts as the cache holds them.
        totals = [n + steps for n in contexts]
        k, v = (dev.alloc(2 * sum(totals) * KV_ROW) for _ in range(2))
        read = dev.put(np.concatenate([layer.slots(i, np.arange(n)) for i, n in enumerate(totals)]))
        mlvc_hip.kv_read(layer.cache, mlvc_hip.KvRows(tokens=sum(totals), k=k, v=v, k_stride=KV_ROW, v_stride=KV_ROW, slots=read),
                         dev.stream)
        q = dev.put(np.stack(rotated, 1).reshape(streams * steps, ROW))
        whole = dev.alloc(2 * streams * steps * ROW)
        layer.prompt(q, k, v, (ROW, KV_ROW, KV_ROW), whole, [steps] * streams, totals)
        want = dev.get(whole, (streams * steps, ROW)).astype(np.float64)
        got = np.stack(by_token, 1).reshape(streams * steps, ROW).astype(np.float64)
        return {"contexts": contexts, "steps": steps, "step_us": spent / steps * 1e6, "finite": finite,
                "difference": float(np.linalg.norm(got - want) / np.linalg.norm(want))}
    finally:
        dev.close()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--config", default="codec_enc_1920x1088")
    ap.add_argument("--streams", type=int, default=2)
    ap.add_argument("--frames", type=int, default=2)
    ap.add_argument("--tokens", type=int, default=16)
    a = ap.parse_args()
    r = run(a.config, a.streams, a.frames, a.tokens)
    print(f"contexts of {r['contexts']} tokens, {r['steps']} steps of {r['step_us']:.0f} us; "
          f"step by step against one prompt: relative difference {r['difference']:.2e}")


if __name__ == "__main__":
    main()
