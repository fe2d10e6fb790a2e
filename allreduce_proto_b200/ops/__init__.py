"""Operations: allreduce, its halves, the fused copy/scale/cast kernel, the norm and clipping of gradients, and the
embedding with the gradient of its table."""
from .allreduce import all_gather, allreduce, copy_scale, default_communicator, init, reduce_scatter
from .embedding import embedding, embedding_grad
from .gradients import clip_grad_norm, grad_norm

__all__ = ["allreduce", "reduce_scatter", "all_gather", "copy_scale", "init", "default_communicator", "grad_norm",
           "clip_grad_norm", "embedding", "embedding_grad"]
