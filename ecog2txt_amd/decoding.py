"""Decoding with the trained network (assessment: restore_and_assess, the online predictor): greedy search, beam search and sampling,
one decoder step per token through the launch-per-step kernels; the input projection of a token is a row of a table made once per set of weights.  Mixed into Seq2SeqEngine (engine.py)."""
import ctypes as C

import torch

from .hip_lib import DT_BF16, DT_F32, lib
from .params import EOS_ID, PAD_ID, capture, ceil_div, r8, rk
from .layers import _bf, _f32, _i32
from .serving import sample_config


class DecodingMixin:
    # ------------------------------------------------------------------ decode
    def greedy_decode(self, ws, which='ema', max_len=None, use_graph=False):
        """beam_width 1 decoding (mocha-1_word_sequence.yaml:31); returns int32 [B, L] token ids.
        use_graph: the whole decode of the batch staged in ws -- encoder + L decoder steps of about six launches each -- is
        captured once per (weights, length, input form) and replayed (the shapes are static: every utterance runs all L steps,
        finished ones emit padding); the eager form launches ~6 L + 20 kernels per batch."""
        s = self.spec
        if self._packed != which:
            self.pack(which)
        if use_graph:
            key = ('greedy', which, max_len, bool(ws.get('packed')))
            g = ws['graph'].get(key)
            if g is None:
                self.greedy_decode(ws, which, max_len)                     # warm-up outside the capture
                torch.cuda.synchronize(self.device)
                g = torch.cuda.CUDAGraph()
                with self.on_step_stream():
                    with capture(g):
                        self.greedy_decode(ws, which, max_len)
                g = ws['graph'][key] = (g, ws.get('A_stale'))
            with self.on_step_stream():
                g[0].replay()
            # (a replay runs no host code: the bookkeeping encode() does on the host is restored to what the captured call left --
            #  a replay through the one-pass front-end leaves NO im2row copy of this batch, and a later backward() must know)
            ws['A_stale'] = g[1]
            return ws['hyp']
        src = getattr(self.store, which)
        B, L = ws['B'], ws['L']
        max_len = L if max_len is None else min(max_len, L)
        st = self.stream
        self.encode(ws, src, False)
        lib.e2t_decode_init(ws['done'].data_ptr(), ws['hyp'].data_ptr(), ws['U'].data_ptr(), ws['dlens'].data_ptr(), B, L, EOS_ID, PAD_ID, st)
        dw = ws['dec']
        pw = ws['proj']
        table = self._token_projection_table(src, which)
        if B <= self.small_batch_head_max and self.proj.nl == 1 and self.options['small_batch_head']:
            # ONE or TWO utterances (the online predictor's one, trainers.py:925-949): a step = the recurrence's launch + ONE head
            # launch (e2t_greedy_head_small: projection on the vector units, arg-max, bookkeeping, the next step's input-projection
            # row: 13-14 us) instead of gather + recurrence + a 128-row-tile GEMM for B real rows + arg-max (4.6 + 12.8 + 4.6 us).
            # Measured host to host at cfg2 (profiles/r06_latency_b1.txt): B = 1 0.578 vs 0.620 ms, B = 2 equal, B = 4 0.72 vs 0.66,
            # B = 8 0.90 vs 0.69 -- the kernel takes B <= 8, the engine uses it up to small_batch_head_max = 2
            if self._head_scratch is None:
                self._head_scratch = torch.zeros(2 + 2 * 64 * 8, dtype=torch.int32, device=self.device)
            lib.e2t_gather_rows_u32(table.data_ptr(), ws['U'].data_ptr(), B, B, self.dec.N4 // 2, dw['Gx'].data_ptr(), st)
            pr = self.proj
            for l in range(max_len):
                self.dec.fwd(dw, None, ws['dlens'], src, False, c0=ws['c0'], steps=(l, l + 1))
                more = l + 1 < max_len
                lib.e2t_greedy_head_small(dw['Yext'].data_ptr() + 2 * (l + 1) * B * self.dec.ldy, self.dec.ldy, pr.WT[0].data_ptr(), pr.in_ld,
                                          pr.bias_ptr(0, src), B, s.vocab, s.dec_rnn, l, L, EOS_ID, PAD_ID, ws['done'].data_ptr(),
                                          ws['hyp'].data_ptr(), ws['U'].data_ptr() + 4 * (l + 1) * B if l + 1 < L else None,
                                          table.data_ptr() if more else None, self.dec.N4 // 2,
                                          dw['Gx'].data_ptr() + 2 * (l + 1) * B * self.dec.N4 if more else None,
                                          self._head_scratch.data_ptr(), st)
            return ws['hyp']
        for l in range(max_len):
            # input projection of this step's tokens: rows of the table (embedding and projection of a token are the same for every
            # utterance and step -- decoding applies no dropout: the embedding lookup + a 256-row GEMM per step were two launches)
            lib.e2t_gather_rows_u32(table.data_ptr(), ws['U'].data_ptr() + 4 * l * B, B, B, self.dec.N4 // 2,
                                    dw['Gx'].data_ptr() + 2 * l * B * self.dec.N4, st)
            self.dec.fwd(dw, None, ws['dlens'], src, False, c0=ws['c0'], steps=(l, l + 1))
            # logits for this step: run the projection stack on rows [l*B, (l+1)*B) of the ext array (t+1 block)
            self._proj_rows(ws, src, l)
            nxt = ws['U'].data_ptr() + 4 * (l + 1) * B if l + 1 < L else None
            lib.e2t_greedy_step(pw['out'].data_ptr() + 4 * l * B * s.vocab, s.vocab, B, s.vocab, l, L, EOS_ID, PAD_ID,
                                ws['done'].data_ptr(), ws['hyp'].data_ptr(), nxt, st)
        return ws['hyp']

    def sample_decode(self, ws, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, which='ema', max_len=None, int8_projection=False,
                      use_graph=False):
        """Draws the words of the batch staged in ws instead of taking the arg-max: (int32 [B, L] token ids, fp32 [B] sums of the drawn
        words' log-probabilities among the kept ones).  u: fp32 [steps, B] uniform numbers in [0, 1) on the engine's device, one a
        word: the same numbers draw the same words.  temperature, top_k, top_p, min_p as in e2t_sample_rows (include/ecog2txt_hip.h),
        numbers or device tensors of B (one an utterance); temperature 0 gives greedy_decode's words.
        int8_projection: the vocabulary projection with 8-bit weights (a scale a word) and states (a scale an utterance and step).
        use_graph: as in greedy_decode; one graph serves every u and all settings.  Both results are the workspace's own arrays."""
        s = self.spec
        B, L = ws['B'], ws['L']
        max_len = L if max_len is None else min(max_len, L)
        sm = self._sample_buffers(ws)
        if not isinstance(u, torch.Tensor) or u.dtype is not torch.float32 or u.device != sm['u'].device or u.dim() != 2 or u.shape[0] < max_len or u.shape[1] != B:
            raise ValueError('sample_decode: u must be float32 [>= %d, %d] on %s' % (max_len, B, sm['u'].device))
        for name, v in (('temperature', temperature), ('top_k', top_k), ('top_p', top_p), ('min_p', min_p)):
            if isinstance(v, torch.Tensor):
                if v.shape != (B,) or v.device != sm['u'].device:
                    raise ValueError('sample_decode: %s must be a number or a tensor of %d on %s' % (name, B, sm['u'].device))
                v = v.detach()
                sm[name].copy_(v.clamp(-1, 2 ** 31 - 1) if name == 'top_k' and v.dtype is torch.int64 else v)
            else:
                sm[name].fill_(max(-1, min(int(v), 2 ** 31 - 1)) if name == 'top_k' else float(v))
        sm['u'][:max_len].copy_(u[:max_len].detach())
        if self._packed != which:
            self.pack(which)
        if not use_graph:
            self._sample_steps(ws, which, max_len, int8_projection)
            return ws['hyp'], sm['score']
        key = ('sample', which, max_len, bool(ws.get('packed')), bool(int8_projection))
        g = ws['graph'].get(key)
        if g is None:
            self._sample_steps(ws, which, max_len, int8_projection)        # warm-up outside the capture
            torch.cuda.synchronize(self.device)
            g = torch.cuda.CUDAGraph()
            with self.on_step_stream():
                with capture(g):
                    self._sample_steps(ws, which, max_len, int8_projection)
            g = ws['graph'][key] = (g, ws.get('A_stale'))
        with self.on_step_stream():
            g[0].replay()
        ws['A_stale'] = g[1]                                               # (what encode() notes on the host: greedy_decode)
        return ws['hyp'], sm['score']

    def _sample_buffers(self, ws):
        """What a captured sample_decode reads and writes at fixed places: uniforms, settings, score, scratch."""
        sm = ws.get('sample')
        if sm is None:
            B, L, dev = ws['B'], ws['L'], self.device
            sm = ws['sample'] = dict(u=_f32(L, B, device=dev), score=_f32(B, device=dev), temperature=_f32(B, device=dev), top_p=_f32(B, device=dev),
                                     min_p=_f32(B, device=dev), top_k=_i32(B, device=dev))
            need = lib.e2t_sample_ws_bytes(B, self.spec.vocab)
            sm['ws'] = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        return sm

    def _sample_steps(self, ws, which, max_len, int8):
        s = self.spec
        src = getattr(self.store, which)
        B, L = ws['B'], ws['L']
        st = self.stream
        dw, pw, sm = ws['dec'], ws['proj'], ws['sample']
        cfg = sample_config(B, sm['u'].get_device(), sm['temperature'], sm['top_k'], sm['top_p'], sm['min_p'])
        self.encode(ws, src, False)
        lib.e2t_decode_init(ws['done'].data_ptr(), ws['hyp'].data_ptr(), ws['U'].data_ptr(), ws['dlens'].data_ptr(), B, L, EOS_ID, PAD_ID, st)
        lib.e2t_fill_u32(sm['score'].data_ptr(), B, 0, st)
        table = self._token_projection_table(src, which)
        q8 = self._projection_i8(which) if int8 else None
        for l in range(max_len):
            lib.e2t_gather_rows_u32(table.data_ptr(), ws['U'].data_ptr() + 4 * l * B, B, B, self.dec.N4 // 2,
                                    dw['Gx'].data_ptr() + 2 * l * B * self.dec.N4, st)
            self.dec.fwd(dw, None, ws['dlens'], src, False, c0=ws['c0'], steps=(l, l + 1))
            self._proj_rows(ws, src, l, q8)
            lib.e2t_sample_step(pw['out'].data_ptr() + 4 * l * B * s.vocab, DT_F32, s.vocab, B, s.vocab, sm['u'].data_ptr() + 4 * l * B, C.byref(cfg),
                                l, L, EOS_ID, PAD_ID, ws['done'].data_ptr(), ws['hyp'].data_ptr(),
                                ws['U'].data_ptr() + 4 * (l + 1) * B if l + 1 < L else None, sm['score'].data_ptr(),
                                sm['ws'].data_ptr() if sm['ws'] is not None else None, sm['ws'].numel() if sm['ws'] is not None else 0, st)

    def beam_decode(self, ws, beam_width, temperature=1.0, which='ema', max_len=None, int8_projection=False):
        """Beam search (`beam_width`, mocha-1_word_sequence.yaml:31; `temperature`, :82) over the batch staged in ws: returns
        (int32 [B, L] token ids of the best hypothesis, fp32 [B, W] scores of the final beams).  The encoder runs once on the
        B utterances; the decoder runs on B x W rows (hypothesis w of utterance b = row b*W + w of a second workspace) with
        the launch-per-step kernels, e2t_beam_step picks the survivors and e2t_beam_reorder moves their state.
        beam_width 1 is greedy_decode (identical tokens); oracle: oracle/seq2seq.py beam_decode.
        int8_projection: as in sample_decode."""
        s = self.spec
        W = int(beam_width)
        assert 1 <= W <= 16
        if self._packed != which:
            self.pack(which)
        src = getattr(self.store, which)
        B, L = ws['B'], ws['L']
        BW = B * W
        max_len = L if max_len is None else min(max_len, L)
        st = self.stream
        wb = self._beam_workspace(ws['sid'], B, W, L)
        if 'beam' not in wb:
            dev = self.device
            wb['beam'] = dict(rep=torch.arange(B, dtype=torch.int32, device=dev).repeat_interleave(W).contiguous(),
                              score=[_f32(BW, device=dev), _f32(BW, device=dev)], done=[_i32(BW, device=dev), _i32(BW, device=dev)],
                              hyp=[_i32(BW, L, device=dev), _i32(BW, L, device=dev)], rowmap=_i32(BW, device=dev),
                              tmp_h=_bf(BW, r8(s.dec_rnn), device=dev), tmp_c=_f32(BW, s.dec_rnn, device=dev),
                              init=torch.tensor([0.0] + [float('-inf')] * (W - 1), dtype=torch.float32, device=dev).repeat(B).contiguous())
        bm = wb['beam']
        self.encode(ws, src, False)
        # every hypothesis starts from the encoder's final state: rows of block 0 of the decoder's ext array and of c0, W times each
        lib.e2t_gather_rows_u32(ws['dec']['Yext'].data_ptr(), bm['rep'].data_ptr(), BW, BW, self.dec.ldy // 2, wb['dec']['Yext'].data_ptr(), st)
        lib.e2t_gather_rows_u32(ws['c0'].data_ptr(), bm['rep'].data_ptr(), BW, BW, s.dec_rnn, wb['c0'].data_ptr(), st)
        bm['score'][0].copy_(bm['init'])                          # beam 0: score 0, the others -inf (W copies of one state)
        lib.e2t_fill_u32(bm['done'][0].data_ptr(), BW, 0, st)
        lib.e2t_fill_u32(bm['hyp'][0].data_ptr(), BW * L, PAD_ID, st)
        lib.e2t_fill_u32(wb['U'].data_ptr(), BW, EOS_ID, st)
        lib.e2t_fill_u32(wb['dlens'].data_ptr(), BW, L, st)
        dw, pw = wb['dec'], wb['proj']
        table = self._token_projection_table(src, which)
        q8 = self._projection_i8(which) if int8_projection else None
        RT, UT = ceil_div(BW, 16), ceil_div(s.dec_rnn, 16)
        cs_step = RT * UT * 2 * 64 * 2                            # floats of one step's lane-native cell save
        cur = 0
        for l in range(max_len):
            lib.e2t_gather_rows_u32(table.data_ptr(), wb['U'].data_ptr() + 4 * l * BW, BW, BW, self.dec.N4 // 2,
                                    dw['Gx'].data_ptr() + 2 * l * BW * self.dec.N4, st)
            self.dec.fwd(dw, None, wb['dlens'], src, False, c0=wb['c0'], steps=(l, l + 1))
            self._proj_rows(wb, src, l, q8)
            nxt = wb['U'].data_ptr() + 4 * (l + 1) * BW if l + 1 < L else None
            lib.e2t_beam_step(pw['out'].data_ptr() + 4 * l * BW * s.vocab, s.vocab, B, W, s.vocab, float(temperature), l, L, EOS_ID, PAD_ID,
                              bm['score'][cur].data_ptr(), bm['done'][cur].data_ptr(), bm['hyp'][cur].data_ptr(),
                              bm['score'][1 - cur].data_ptr(), bm['done'][1 - cur].data_ptr(), bm['hyp'][1 - cur].data_ptr(),
                              bm['rowmap'].data_ptr(), nxt, st)
            cur = 1 - cur
            if l + 1 < max_len:
                lib.e2t_beam_reorder(dw['Yext'].data_ptr() + 2 * (l + 1) * BW * self.dec.ldy, self.dec.ldy,
                                     dw['Cs'].data_ptr() + 4 * l * cs_step, BW, s.dec_rnn, bm['rowmap'].data_ptr(),
                                     bm['tmp_h'].data_ptr(), bm['tmp_c'].data_ptr(), st)
        hyp = bm['hyp'][cur].view(B, W, L)[:, 0, :].contiguous()  # survivors are kept best first
        return hyp, bm['score'][cur].view(B, W)

    def _token_projection_table(self, src, which=None):
        """bf16 [V][4 H_d]: the decoder's input projection of every token, W_x . embedding[v] + b, from the images packed last
        (one 1806-row GEMM per decode call in place of an embedding lookup + a B-row GEMM per step: the same operands and K
        order; bit-identical to the per-step product where the launch plan picks the same tile and K split for M = V as for
        M = B -- it does at the tested shapes, tests/test_gpu_kernels.py -- and within fp32 round-off of one bf16 ulp elsewhere)."""
        s = self.spec
        if self._dec_table is None:
            self._dec_table = _bf(s.vocab, self.dec.N4, device=self.device)
        # (round 6: the table depends on the weights only -- it is made once per set of operand images, not once per call: 12 us of a
        #  0.6-ms single-utterance decode.  _img_version moves whenever an image or a parameter may have changed.)
        key = (which, self._img_version) if which is not None else None
        if torch.cuda.is_current_stream_capturing():
            key = None                 # (a captured decode rebuilds the table at every replay: the graph outlives the weights it was captured with)
        if key is not None and self._dec_table_key == key:
            return self._dec_table
        self._dec_table_key = key
        self.gemm(self.emb.data_ptr(), self.E8, self.dec.WxT.data_ptr(), self.E8, self._dec_table.data_ptr(), self.dec.N4,
                  s.vocab, self.dec.N4, self.E8, bias=self.dec.bias_ptr(src), out_bf16=True)
        return self._dec_table

    def _beam_workspace(self, sid, B, W, L):
        """The decoder-side arrays of B x W hypothesis rows, and nothing else: a full training workspace of B x W rows would
        also hold the inputs, the im2row copy and every encoder layer's activations and gradients W times over (tens of GB at
        beam_width 16), and its cache key could alias a live training workspace of the same row count."""
        key = ('beam', sid, B, W, L)
        wb = self._ws.get(key)
        if wb is None:
            s, dev = self.spec, self.device
            BW = B * W
            Md = L * BW
            wb = dict(sid=sid, B=BW, L=L, Md=Md, enc=[], graph={})
            wb['U'] = _i32(Md, device=dev)
            wb['e'] = _bf(Md, self.E8, device=dev)
            wb['dec'] = self.dec.alloc(L, BW)
            wb['c0'] = _f32(BW, s.dec_rnn, device=dev)
            wb['dlens'] = _i32(BW, device=dev)
            wb['proj'] = self.proj.alloc(Md)
            self._ws[key] = wb
        return wb

    def _projection_i8(self, which):
        """(int8 [V][K up to 64], fp32 [V]): the vocabulary projection's packed bf16 weights in 8 bits, made once per set of operand images
        like the token table (a captured decode makes them anew at every replay).  K = the layer's real inputs: the ones column
        that carries the bias in the state rows stays out, the bias is added in fp32."""
        pr = self.proj
        K, V = pr.sizes[-2], pr.sizes[-1]
        if self._proj_i8 is None:
            self._proj_i8 = (torch.empty(V, rk(K), dtype=torch.int8, device=self.device), _f32(V, device=self.device))
        key = None if torch.cuda.is_current_stream_capturing() else (which, self._img_version)
        if key is None or self._proj_i8_key != key:
            q, scale = self._proj_i8
            lib.e2t_quant_rows_i8(pr.WT[-1].data_ptr(), DT_BF16, pr.WT[-1].shape[1], V, K, q.data_ptr(), q.shape[1], scale.data_ptr(), self.stream)
            self._proj_i8_key = key
        return self._proj_i8

    def _proj_rows(self, ws, src, l, q8=None):
        """Projection stack on decoder step l (un-dropped h_t = ext block l+1).  q8: the last layer's weights in 8 bits (_projection_i8)."""
        s = self.spec
        B = ws['B']
        pr, pw = self.proj, ws['proj']
        cur = ws['dec']['Yext'].data_ptr() + 2 * (l + 1) * B * self.dec.ldy
        ld = self.dec.ldy
        for i in range(pr.nl):
            last = i == pr.nl - 1
            fout = pr.sizes[i + 1]
            kin = pr.in_ld if i == 0 else rk(pr.sizes[i])
            if last and q8 is not None:
                fin = pr.sizes[i]
                need = lib.e2t_linear_i8_ws_bytes(B, fout, fin)
                if need and 'i8' not in pw:
                    pw['i8'] = torch.empty(need, dtype=torch.uint8, device=self.device)
                lib.e2t_linear_i8(cur, DT_BF16, ld, q8[0].data_ptr(), q8[0].shape[1], q8[1].data_ptr(), pr.bias_ptr(i, src),
                                  pw['out'].data_ptr() + 4 * l * B * fout, fout, B, fout, fin, 0, pw['i8'].data_ptr() if need else None, need, self.stream)
            elif last:
                self.gemm(cur, ld, pr.WT[i].data_ptr(), kin, pw['out'].data_ptr() + 4 * l * B * fout, fout, B, fout, kin,
                          bias=pr.bias_ptr(i, src))
            else:
                o = pw['act'][i].data_ptr() + 2 * l * B * rk(fout)
                self.gemm(cur, ld, pr.WT[i].data_ptr(), kin, o, rk(fout), B, fout, kin, bias=pr.bias_ptr(i, src),
                          relu=True, out_bf16=True)
                cur, ld = o, rk(fout)
