"""Single-GPU prefill, cached decode and greedy Qwen3 generation on HIP kernels."""
from .model import CapturedGreedyRequest, DecodeSession, Int8KVCache, KVCache, SharedPrefixCache, TritonQwen3Inference

__all__ = ['KVCache', 'Int8KVCache', 'SharedPrefixCache', 'TritonQwen3Inference', 'CapturedGreedyRequest', 'DecodeSession']
