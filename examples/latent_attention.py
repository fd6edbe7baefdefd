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

Needs the built libraries, torch and an MI355X.
"""

from __future__ import annotations

import argparse
import ctypes as C
import pathlib
import sys
import tempfile
import time

import numpy as np
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "mlvc.cpp_amd" / "python"))

import mlvc_hip  # noqa: E402

Q_HEADS, KV_HEADS, DIM, PAGE = 16, 4, 64, 64
SCALE, EPS = DIM ** -0.5, 1e-6


def encode(config: str, streams: int, frames: int) -> list[torch.Tensor]:
    """Latents of each stream's frames as tokens [frames * h * w, channels]; stream i has i frames fewer, one at least."""
    out = []
    with tempfile.TemporaryDirectory() as d:
        mlvc_hip.synth_write(config, d, 0)
        bindings, _ = mlvc_hip.synth_bindings(config)
        with mlvc_hip.Backend(d, "hip", device_id=0) as graph:
            graph.load("MLVCEncoder", bindings)
            for stream in range(streams):
                graph.reset_state()
                tokens = []
                for frame in range(max(1, frames - stream) + 1):  # and the frame to come
                    inputs = [np.array([32], np.int32) if t == np.int32 else
                              mlvc_hip.synth_input(config, i, frame, s, seed=stream)
                              for i, (s, t) in enumerate(zip(graph.in_shapes, graph.in_dtypes))]
                    y = graph.run(inputs)[0].view(np.float16)[0]
                    tokens.append(y.reshape(y.shape[0], -1).T)
                out.append(torch.from_numpy(np.ascontiguousarray(np.concatenate(tokens))).cuda())
    return out


def _i32(values) -> torch.Tensor:
    return torch.as_tensor(np.asarray(values, np.int32)).cuda()


class Layer:
    """One attention layer and the cache of its streams."""

    def __init__(self, channels: int, contexts: list[int], room: int):
        g = torch.Generator().manual_seed(1)
        width = (Q_HEADS + 2 * KV_HEADS) * DIM
        self.w_in = (torch.randn(channels, width, generator=g) / channels ** 0.5).half().cuda()
        self.norm_q, self.norm_k = ((1 + 0.1 * torch.randn(DIM, generator=g)).half().cuda() for _ in range(2))
        freqs, self.rot_scale = mlvc_hip.rope_frequencies(DIM, 10000.0, mlvc_hip.ROPE_BANDS, 4.0, 8160)
        self.freqs = torch.from_numpy(freqs).cuda()
        # Every stream gets the pages of its context and of the tokens to come.
        pages = [-(-(n + room) // PAGE) for n in contexts]
        order = torch.randperm(sum(pages), generator=g).tolist()
        self.table = np.full((len(pages), max(pages)), -1, np.int32)
        for i, n in enumerate(pages):
            self.table[i, :n] = [order.pop() for _ in range(n)]
        self.device_table = _i32(self.table)
        self.cache = mlvc_hip.KvCache(kind=mlvc_hip.KV_INT8, pages=sum(pages), page_size=PAGE, heads=KV_HEADS, head_dim=DIM)
        values, scales = mlvc_hip.kv_cache_bytes(self.cache)
        self.memory = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (values, values, scales, scales)]
        self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale = (m.data_ptr() for m in self.memory)

    def slots(self, stream: int, positions) -> np.ndarray:
        p = np.asarray(positions)
        return self.table[stream, p // PAGE] * PAGE + p % PAGE

    def parts(self, qkv: torch.Tensor):
        """Addresses of q, k and v in rows of the projection, and the rows' stride."""
        at = qkv.data_ptr()
        return at, at + 2 * Q_HEADS * DIM, at + 2 * (Q_HEADS + KV_HEADS) * DIM, qkv.shape[1]

    def rotate_and_keep(self, qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, stream: int) -> None:
        q, k, v, stride = self.parts(qkv)
        mlvc_hip.qk_norm_rope(mlvc_hip.QkNormRope(
            tokens=qkv.shape[0], q_heads=Q_HEADS, k_heads=KV_HEADS, head_dim=DIM, q=q, k=k, q_out=q, k_out=k,
            q_stride=stride, k_stride=stride, q_out_stride=stride, k_out_stride=stride, q_weight=self.norm_q.data_ptr(),
            k_weight=self.norm_k.data_ptr(), eps=EPS, positions=positions.data_ptr(), freqs=self.freqs.data_ptr(),
            rot_dim=DIM, interleaved=0, rot_scale=self.rot_scale), stream)
        mlvc_hip.kv_write(self.cache, mlvc_hip.KvRows(tokens=qkv.shape[0], k=k, v=v, k_stride=stride, v_stride=stride,
                                                      slots=slots.data_ptr()), stream)

    def prompt(self, q, k, v, strides, out: torch.Tensor, queries: list[int], keys: list[int]) -> None:
        starts_q, starts_k = (_i32(np.concatenate([[0], np.cumsum(n)])) for n in (queries, keys))
        mlvc_hip.attention_prompt(mlvc_hip.PromptAttention(
            sequences=len(queries), q_heads=Q_HEADS, kv_heads=KV_HEADS, head_dim=DIM, q=q, k=k, v=v, out=out.data_ptr(),
            q_stride=strides[0], k_stride=strides[1], v_stride=strides[2], out_stride=Q_HEADS * DIM,
            q_starts=starts_q.data_ptr(), k_starts=starts_k.data_ptr(), q_tokens=sum(queries), k_tokens=sum(keys),
            longest_q=max(queries), causal=1, scale=SCALE), torch.cuda.current_stream().cuda_stream)


def run(config: str = "codec_enc_1920x1088", streams: int = 2, frames: int = 2, steps: int = 16) -> dict:
    latents = encode(config, streams, frames)
    per_frame = latents[0].shape[0] // (max(1, frames) + 1)
    contexts = [t.shape[0] - per_frame for t in latents]
    steps = min(steps, per_frame)
    layer = Layer(latents[0].shape[1], contexts, steps)

    # The frames that are there: one packed prompt.
    qkv = torch.cat([t[:n] for t, n in zip(latents, contexts)]) @ layer.w_in
    positions = _i32(np.concatenate([np.arange(n) for n in contexts]))
    slots = _i32(np.concatenate([layer.slots(i, np.arange(n)) for i, n in enumerate(contexts)]))
    out = torch.empty(qkv.shape[0], Q_HEADS * DIM, dtype=torch.float16, device="cuda")
    layer.rotate_and_keep(qkv, positions, slots, torch.cuda.current_stream().cuda_stream)
    q, k, v, stride = layer.parts(qkv)
    layer.prompt(q, k, v, (stride,) * 3, out, contexts, contexts)

    # The next frame, token by token: the step's buffers stay, so it is captured once.
    lib = mlvc_hip.device_lib()
    stream, graph = C.c_void_p(), C.c_void_p()

    def check(rc):
        if rc != 0:
            raise mlvc_hip.MlvcError(lib.mlvc_hip_last_error().decode())

    check(lib.mlvc_hip_stream_create(C.byref(stream)))
    mine = torch.cuda.ExternalStream(stream.value)
    mine.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(mine):
        row = torch.empty(streams, qkv.shape[1], dtype=torch.float16, device="cuda")
        step_out = torch.empty(streams, Q_HEADS * DIM, dtype=torch.float16, device="cuda")
        at, slot, lengths = (torch.zeros(streams, dtype=torch.int32, device="cuda") for _ in range(3))
        attend = mlvc_hip.TokenAttention(
            cache=C.pointer(layer.cache), streams=streams, q_heads=Q_HEADS, q=row.data_ptr(), out=step_out.data_ptr(),
            q_stride=row.shape[1], out_stride=Q_HEADS * DIM, table=layer.device_table.data_ptr(),
            table_stride=layer.table.shape[1], lengths=lengths.data_ptr(), longest=max(contexts) + steps, scale=SCALE)
        need = mlvc_hip.attention_token_workspace_bytes(attend)
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        attend.workspace, attend.workspace_bytes = workspace.data_ptr(), need
        torch.cuda.synchronize()
        check(lib.mlvc_hip_capture_begin(stream))
        layer.rotate_and_keep(row, at, slot, stream)
        mlvc_hip.attention_token(attend, stream)
        check(lib.mlvc_hip_capture_end(stream, C.byref(graph)))

        by_token, projected = [], []
        began = time.perf_counter()
        for step in range(steps):
            row.copy_(torch.stack([t[n + step] for t, n in zip(latents, contexts)]) @ layer.w_in)
            at.copy_(_i32([n + step for n in contexts]))
            slot.copy_(_i32([layer.slots(i, n + step) for i, n in enumerate(contexts)]))
            lengths.copy_(at + 1)
            check(lib.mlvc_hip_graph_launch(graph, stream))
            by_token.append(step_out.clone())
            projected.append(row.clone())
        mine.synchronize()
        step_us = (time.perf_counter() - began) / steps * 1e6
    check(lib.mlvc_hip_graph_destroy(graph))
    torch.cuda.current_stream().wait_stream(mine)

    # The same tokens as one prompt on the contexts as the cache holds them.
    totals = [n + steps for n in contexts]
    read = _i32(np.concatenate([layer.slots(i, np.arange(n)) for i, n in enumerate(totals)]))
    keys = [torch.empty(sum(totals), KV_HEADS * DIM, dtype=torch.float16, device="cuda") for _ in range(2)]
    here = torch.cuda.current_stream().cuda_stream
    mlvc_hip.kv_read(layer.cache, mlvc_hip.KvRows(tokens=sum(totals), k=keys[0].data_ptr(), v=keys[1].data_ptr(),
                                                  k_stride=KV_HEADS * DIM, v_stride=KV_HEADS * DIM, slots=read.data_ptr()), here)
    queries = torch.stack(projected, 1).reshape(streams * steps, -1)[:, :Q_HEADS * DIM].contiguous()
    whole = torch.empty(streams * steps, Q_HEADS * DIM, dtype=torch.float16, device="cuda")
    layer.prompt(queries.data_ptr(), keys[0].data_ptr(), keys[1].data_ptr(), (Q_HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM),
                 whole, [steps] * streams, totals)
    torch.cuda.synchronize()
    check(lib.mlvc_hip_stream_destroy(stream))
    got = torch.stack(by_token, 1).reshape(streams * steps, -1).float()
    difference = (got - whole.float()).norm() / whole.float().norm()
    return {"contexts": contexts, "steps": steps, "step_us": step_us, "difference": difference.item(),
            "finite": bool(torch.isfinite(out).all() and torch.isfinite(got).all())}


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
